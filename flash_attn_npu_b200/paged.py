"""Paged key/value cache: writing new tokens, reading tokens back, attention over it, also behind prefixes
that sequences share; the attention weight that each token received, and eviction by it.

For serving, where sequences of unequal lengths keep their keys and values from call to call.
Sequences share caches of pages,

    k_cache, v_cache   [num_pages, heads_kv, page_size, head_dim]   fp16, bf16 or float8_e4m3fn
    k_scale, v_scale   [num_pages, heads_kv, page_size] float32, with a float8 cache only
    page_table         [seqs, columns] int32: the pages of each sequence, in order
    kv_lens            [seqs] int32: its length in the cache, its new tokens included
    offsets            [seqs + 1] int32: its rows in the packed tensors of new tokens

Row i of sequence b is row offsets[b] + i of the packed tensors [total, heads, head_dim], and the
token at position kv_lens[b] - (offsets[b + 1] - offsets[b]) + i of the sequence.  A decoding step
has one row per sequence (offsets = 0, 1, 2, ...), a prompt or a chunk of one has many; a call may
mix them.  Packed rows of no sequence (behind offsets[-1], or before offsets[0]) are padding: what
they hold does not matter, and outputs there are left as they were.  Pages behind a sequence's length
may hold anything, NaN included.

A float8 cache holds code = round_e4m3(x / scale) with one power of two per (token, kv head); any
positive, normal scale can be read.  page_size is a power of two, 8 .. 1024.  Two sequences may share
pages (a common prefix), but a call to `write` must not be given the same place twice: which of the
rows stays there is open.

`page_table`, `kv_lens` and `offsets` (which do not decrease) are device data, which a launch does not
wait for: a kernel on another stream must not change them while a call runs.  Entries outside the cache
or the table are never followed: the call reports them through the device status word
(`ops.check_device_status` raises), and the results of that sequence are undefined.
"""
from __future__ import annotations

import ctypes
import math
import operator

import torch

from . import _native, ops

FP8 = torch.float8_e4m3fn
_CACHE_CODES = {torch.float16: _native.FA_DTYPE_FP16, torch.bfloat16: _native.FA_DTYPE_BF16,
                FP8: _native.FA_DTYPE_FP8_E4M3}
_ROW_CODES = {torch.float16: _native.FA_DTYPE_FP16, torch.bfloat16: _native.FA_DTYPE_BF16}


def empty_cache(num_pages: int, page_size: int, heads_kv: int, head_dim: int, dtype=torch.bfloat16,
                device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of these sizes, not initialised; the scales are None
    unless dtype is float8_e4m3fn."""
    shape = (num_pages, heads_kv, page_size, head_dim)
    k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype != FP8:
        return k, v, None, None
    return k, v, *(torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2))


# ------------------------------------------------------------------------------------- checks
def validate_cache(k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale) -> None:
    """Shapes, types and layout of a cache and its sequences, on tensors of any device (`offsets` None:
    a call without packed rows)."""
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape [num_pages, heads_kv, "
                         "page_size, head_dim]")
    if k_cache.dtype != v_cache.dtype or k_cache.dtype not in _CACHE_CODES:
        raise ValueError("k_cache and v_cache must both be float16, bfloat16 or float8_e4m3fn")
    pages, heads, size, head_dim = k_cache.shape
    if head_dim not in ops.HEAD_DIMS:
        raise ValueError("HEAD_DIM must be one of {16, 32, 64, 128, 256}")
    if not 8 <= size <= 1024 or size & (size - 1):
        raise ValueError("page_size must be a power of two, 8 .. 1024")
    if pages < 1 or heads < 1:
        raise ValueError("a cache needs at least one page and one head")
    if pages > 1 << 30 or heads > 65536:
        raise ValueError("a cache has at most 2^30 pages and 65536 heads")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not _aligned(t):
            raise ValueError(f"{name} needs a unit inner stride and 16-byte aligned strides")
        if any(t.shape[d] > 1 and t.stride(d) >= 1 << 38 for d in range(3)):
            raise ValueError(f"{name} needs strides below 2^38")
    if (k_scale is None) != (v_scale is None) or (k_scale is None) == (k_cache.dtype == FP8):
        raise ValueError("k_scale and v_scale go with a float8_e4m3fn cache, and with no other")
    if k_scale is not None:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.shape != k_cache.shape[:3] or t.dtype != torch.float32:
                raise ValueError(f"{name} must be float32 [num_pages, heads_kv, page_size]")
            if not _aligned(t):
                raise ValueError(f"{name} needs a unit inner stride and 16-byte aligned strides")
    validate_sequences(page_table, offsets, kv_lens, size)
    for t in (k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale):
        if t is not None and t.device != k_cache.device:
            raise ValueError("all tensors of a paged call must be on the same device")
        if t is not None and t.is_neg():
            raise ValueError("a cache, its scales and its sequences must not be negated views")


def validate_sequences(page_table, offsets, kv_lens, page_size,
                       names=("page_table", "offsets", "kv_lens"), rows="seqs") -> None:
    """Shapes, types and layout of a page table and what goes with it."""
    table, offs, lens = names
    if offsets is None:
        offsets = kv_lens.new_empty(kv_lens.shape[0] + 1 if kv_lens.ndim == 1 else 0, dtype=torch.int32)
    if (page_table.ndim != 2 or offsets.ndim != 1 or kv_lens.ndim != 1
            or offsets.shape[0] != page_table.shape[0] + 1
            or kv_lens.shape[0] != page_table.shape[0]):
        raise ValueError(f"{table} must be [{rows}, columns], {offs} [{rows} + 1], {lens} [{rows}]")
    if any(t.dtype != torch.int32 for t in (page_table, offsets, kv_lens)):
        raise ValueError(f"{table}, {offs} and {lens} must be int32")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1 or not (
            offsets.is_contiguous() and kv_lens.is_contiguous()):
        raise ValueError(f"{offs}, {lens} and the rows of {table} must be contiguous")
    if page_table.shape[1] * page_size > 1 << 30:
        raise ValueError(f"{table} names more than 2^30 positions a sequence")


def _validate_rows(name, t, k_cache, heads) -> None:
    if t.ndim != 3 or t.shape[1] != heads or t.shape[2] != k_cache.shape[3]:
        raise ValueError(f"{name} must be [total, heads, head_dim] with the cache's head_dim and "
                         f"{heads} heads (got {tuple(t.shape)})")
    if t.dtype not in _ROW_CODES or k_cache.dtype not in (t.dtype, FP8):
        raise ValueError(f"{name} must be float16 or bfloat16, and of the cache's type unless that "
                         "is float8_e4m3fn")
    if t.device != k_cache.device:
        raise ValueError("all tensors of a paged call must be on the same device")
    if t.shape[0] > 1 << 30:
        raise ValueError(f"{name} has more than 2^30 rows")


def validate_attention(q, k_cache, v_cache, page_table, offsets, kv_lens, k_scale=None,
                       v_scale=None, max_q_len=None) -> None:
    """The rules of `attention`, on tensors of any device."""
    validate_cache(k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
    heads_kv = k_cache.shape[1]
    if q.ndim != 3 or q.shape[1] == 0 or q.shape[1] % heads_kv:
        raise ValueError("q must be [total, heads_q, head_dim], heads_q a multiple of heads_kv")
    _validate_rows("q", q, k_cache, q.shape[1])
    if q.shape[1] > 32768:
        raise ValueError("q has more than 32768 heads")
    if q.shape[0] * q.shape[1] > (1 << 30) - 1:
        raise ValueError("q has more than 2^30 - 1 (token, head) rows")
    if max_q_len is not None and max_q_len < 0:
        raise ValueError("max_q_len must not be negative")


def validate_prefix_attention(q, k_cache, v_cache, prefix_table, prefix_offsets, prefix_lens, page_table,
                              offsets, kv_lens, k_scale=None, v_scale=None, max_q_len=None,
                              max_prefix_q_len=None) -> None:
    """The rules of `prefix_attention`, on tensors of any device."""
    validate_attention(q, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale, max_q_len)
    prefix = (prefix_table, prefix_offsets, prefix_lens)
    validate_sequences(*prefix, k_cache.shape[2], ("prefix_table", "prefix_offsets", "prefix_lens"),
                       "prefixes")
    if any(t.device != k_cache.device for t in prefix):
        raise ValueError("all tensors of a paged call must be on the same device")
    if any(t.is_neg() for t in prefix):
        raise ValueError("a cache, its scales and its sequences must not be negated views")
    if max_prefix_q_len is not None and max_prefix_q_len < 0:
        raise ValueError("max_prefix_q_len must not be negative")


def _validate_weights(weights, k_cache) -> None:
    if weights.shape != k_cache.shape[:3] or weights.dtype != torch.float32:
        raise ValueError("weights must be float32 [num_pages, heads_kv, page_size]")
    if not _aligned(weights):
        raise ValueError("weights needs a unit inner stride and 16-byte aligned strides")
    if weights.device != k_cache.device:
        raise ValueError("all tensors of a paged call must be on the same device")
    if weights.is_neg():
        raise ValueError("weights must not be a negated view")


def validate_attention_weights(q, lse, k_cache, page_table, offsets, kv_lens, weights, k_scale=None,
                               max_q_len=None) -> None:
    """The rules of `attention_weights`, on tensors of any device."""
    if (k_scale is None) == (k_cache.dtype == FP8):
        raise ValueError("k_scale goes with a float8_e4m3fn cache, and with no other")
    validate_attention(q, k_cache, k_cache, page_table, offsets, kv_lens, k_scale, k_scale, max_q_len)
    _validate_weights(weights, k_cache)
    if lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError("lse must be float32 [total, heads_q]")


def validate_evict(k_cache, v_cache, weights, page_table, kv_lens, keep, recent, k_scale=None, v_scale=None,
                   to_table=None) -> None:
    """The rules of `evict`, on tensors of any device."""
    validate_cache(k_cache, v_cache, page_table, None, kv_lens, k_scale, v_scale)
    _validate_weights(weights, k_cache)
    if not 0 <= recent <= keep <= 1 << 30:
        raise ValueError("keep and recent must be 0 <= recent <= keep <= 2^30")
    if page_table.shape[0] * k_cache.shape[1] > 1 << 24:
        raise ValueError("an eviction takes at most 2^24 heads of sequences")
    if to_table is not None:
        if to_table.ndim != 2 or to_table.shape[0] != page_table.shape[0] or to_table.dtype != torch.int32:
            raise ValueError("to_table must be int32 [seqs, columns]")
        if to_table.shape[1] > 1 and to_table.stride(1) != 1:
            raise ValueError("the rows of to_table must be contiguous")
        if to_table.shape[1] * k_cache.shape[2] > 1 << 30:
            raise ValueError("to_table names more than 2^30 positions a sequence")
        if to_table.device != k_cache.device:
            raise ValueError("all tensors of a paged call must be on the same device")
        if to_table.is_neg():
            raise ValueError("a cache, its scales and its sequences must not be negated views")


def validate_copy(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale=None,
                  v_scale=None) -> None:
    """The rules of `write` and of `read`'s outputs, on tensors of any device."""
    validate_cache(k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError("k and v must have the same shape and dtype")
    for name, t in (("k", k), ("v", v)):
        _validate_rows(name, t, k_cache, k_cache.shape[1])


def _strided(t) -> bool:
    """Unit inner stride and 16-byte strides."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return False
    return all(t.shape[d] <= 1 or (t.stride(d) > 0 and (t.stride(d) * t.element_size()) % 16 == 0)
               for d in range(t.ndim - 1))


def _aligned(t) -> bool:
    """... and a 16-byte address (of a tensor that has one)."""
    return _strided(t) and (t.device.type == "meta" or hasattr(t, "fake_device")
                            or t.data_ptr() % 16 == 0)


def empty_rows(t):
    """Rows like `t`, not initialised: in its layout where the strides are 16-byte aligned, else
    contiguous (whatever the address, which a traced call does not know)."""
    return torch.empty_like(t) if _strided(t) else t.new_empty(t.shape)


def _require_cuda(t) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"paged calls take CUDA tensors on an sm_100 device (got {t.device})")


# ------------------------------------------------------------------------------------ launching
# A call goes to the native binding first, which does the checks above on the tensors themselves.
# What it hands back (None) is looked at here: refused with a reason, or prepared and called again.
_binding = None
_PREPARED: set[int] = set()  # devices whose status word the binding knows


def _native_binding():
    global _binding
    if _binding is None:
        try:
            from . import _paged_binding
        except ImportError as exc:
            raise RuntimeError(f"the paged calls need {exc.name or '_paged_binding'}; build it with "
                               "`python -m flash_attn_npu_b200.build`") from None
        lib = _native.load()
        def addresses(*calls):
            return (ctypes.cast(fn, ctypes.c_void_p).value for fn in calls)

        _paged_binding.setup(*addresses(
            lib.fa_paged_attn_sm100, lib.fa_paged_workspace_bytes, lib.fa_paged_write_sm100,
            lib.fa_paged_read_sm100))
        _paged_binding.setup_more(*addresses(
            lib.fa_paged_prefix_sm100, lib.fa_paged_prefix_workspace_bytes, lib.fa_paged_weights_sm100,
            lib.fa_paged_weights_workspace_bytes, lib.fa_paged_evict_sm100,
            lib.fa_paged_evict_workspace_bytes))
        _binding = _paged_binding
    return _binding


def _call(name, device, *args):
    """Call the binding once its device is prepared."""
    binding = _native_binding()
    index = ops._device_index(device)
    if index in _PREPARED:
        res = getattr(binding, name)(*args)
    elif index in ops._STATUS_WORDS or not torch.cuda.is_current_stream_capturing():
        binding.set_status(index, ops.device_status_word(device).data_ptr(), True)
        _PREPARED.add(index)
        res = getattr(binding, name)(*args)
    else:
        # a capture before the device's first launch gets no word: an allocation here would belong
        # to the graph's private pool
        binding.set_status(index, 0, True)
        try:
            res = getattr(binding, name)(*args)
        finally:
            binding.set_status(index, 0, False)
    if res is None:
        raise ValueError("paged calls take dense CUDA tensors with memory of their own, no subclasses")
    return res


def _check(res, device) -> None:
    """Raise for a status code of the library; look at the device's word if that is asked for."""
    if type(res) is int and res != _native.FA_OK:
        exc = _native.NativeError(res, _native.status_string(res))
        if res in (_native.FA_ERR_UNSUPPORTED_HEAD_DIM, _native.FA_ERR_UNSUPPORTED_DTYPE,
                   _native.FA_ERR_INVALID_ARG, _native.FA_ERR_MISALIGNED):
            raise ValueError(str(exc))
        raise exc
    if ops._CHECK_EVERY_CALL:
        ops.check_device_status(device)


def _max_len(n, name="max_q_len"):
    """An upper bound given as any kind of integer, or None."""
    if n is None:
        return None
    try:
        n = operator.index(n)
    except TypeError:
        raise ValueError(f"{name} must be an integer or None (got {n!r})") from None
    return min(n, 1 << 30)  # (there are no more rows)


def _count(n, name) -> int:
    try:
        return operator.index(n)
    except TypeError:
        raise ValueError(f"{name} must be an integer (got {n!r})") from None


def _scale(x) -> float:
    try:
        x = float(x)
    except (TypeError, ValueError):
        raise ValueError(f"sm_scale must be a number (got {x!r})") from None
    if not math.isfinite(ctypes.c_float(x).value):
        raise ValueError(f"sm_scale must be finite in float32 (got {x})")
    return x


def _rows_like(t):
    """`t`, or a copy where its rows are not 16-byte aligned or its memory holds their negatives."""
    return t if _aligned(t) and not t.is_neg() else empty_rows(t).copy_(t.detach())


def _validate_outputs(q, out, lse) -> None:
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype
                            or out.device != q.device or not _aligned(out) or out.is_neg()):
        raise ValueError("out must match q in shape, dtype and device, with a unit inner stride "
                         "and 16-byte aligned strides")
    if lse is not None and (lse.shape != q.shape[:2] or lse.dtype != torch.float32
                            or lse.device != q.device or not lse.is_contiguous() or lse.is_neg()):
        raise ValueError("lse must be a contiguous float32 tensor [total, heads_q]")


def attention(q, k_cache, v_cache, page_table, offsets, kv_lens, causal, sm_scale, k_scale=None,
              v_scale=None, max_q_len=None, out=None, lse=None):
    """Attention of the packed queries q [total, heads_q, head_dim] over the cache; (out, lse).

    Query head h reads kv head h // (heads_q // heads_kv).  Causal: a token attends to positions up
    to its own; else to its whole sequence.  `out` is like q, `lse` [total, heads_q] float32 the
    natural-log logsumexp; a row with no key to attend to gets 0 and -inf.  `max_q_len`: an upper
    bound of a sequence's new tokens that the kernel choice goes by (default: total).  `out` and
    `lse` may be given; rows that belong to no sequence are not written.

    Every value inside a sequence takes part in the products, with a probability of 0 where the
    causal mask hides it: a NaN or an infinity among them may show in any row of the sequence.  Over
    a float8 cache, calls of more than 32 query rows a kv head (`max_q_len` counts) round code *
    scale to q's type: exact for scales that `write` left for rows of that type (up to 63488 in
    float16), else one rounding more, and infinite beyond 65504 with float16 queries.

    Rows that are not 16-byte aligned are copied first.  There is no backward pass: `out` and `lse`
    do not require gradients.
    """
    res = None
    if _binding is not None:
        res = _binding.attention(q, k_cache, v_cache, page_table, offsets, kv_lens, causal, sm_scale,
                                 k_scale, v_scale, max_q_len, out, lse)
    if res is None:
        sm_scale, max_q_len = _scale(sm_scale), _max_len(max_q_len)
        validate_attention(q, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale,
                           max_q_len)
        _require_cuda(q)
        _validate_outputs(q, out, lse)
        res = _call("attention", q.device, _rows_like(q), k_cache, v_cache, page_table, offsets,
                    kv_lens, bool(causal), sm_scale, k_scale, v_scale, max_q_len, out, lse)
    if type(res) is int or ops._CHECK_EVERY_CALL:
        _check(res, q.device)
    return res


def prefix_attention(q, k_cache, v_cache, prefix_table, prefix_offsets, prefix_lens, page_table, offsets,
                     kv_lens, causal, sm_scale, k_scale=None, v_scale=None, max_q_len=None,
                     max_prefix_q_len=None, out=None, lse=None):
    """Attention of sequences that share prefixes, which are read and multiplied once for all; (out, lse).

    Prefix g is the `prefix_lens[g]` tokens in the pages `prefix_table[g]` of the same cache.  The packed
    rows prefix_offsets[g] .. prefix_offsets[g + 1] attend to all of it, and behind it to their own
    sequence: `page_table`, `offsets`, `kv_lens` and `causal` as for `attention`, of the sequences' own
    tokens alone (`kv_lens` does not count the prefix, whose last page no sequence continues).  Rows of no
    group have no prefix, and rows of no sequence are not written.  `lse` is over both.

    `max_prefix_q_len`: an upper bound of the rows that share one prefix, which the kernel choice goes by
    (default: total); `max_q_len`, `out`, `lse` and what values may do as in `attention`.
    """
    res = None
    if _binding is not None:
        res = _binding.prefix_attention(q, k_cache, v_cache, prefix_table, prefix_offsets, prefix_lens,
                                        page_table, offsets, kv_lens, causal, sm_scale, k_scale, v_scale,
                                        max_q_len, max_prefix_q_len, out, lse)
    if res is None:
        sm_scale, max_q_len = _scale(sm_scale), _max_len(max_q_len)
        max_prefix_q_len = _max_len(max_prefix_q_len, "max_prefix_q_len")
        validate_prefix_attention(q, k_cache, v_cache, prefix_table, prefix_offsets, prefix_lens,
                                  page_table, offsets, kv_lens, k_scale, v_scale, max_q_len,
                                  max_prefix_q_len)
        _require_cuda(q)
        _validate_outputs(q, out, lse)
        res = _call("prefix_attention", q.device, _rows_like(q), k_cache, v_cache, prefix_table,
                    prefix_offsets, prefix_lens, page_table, offsets, kv_lens, bool(causal), sm_scale,
                    k_scale, v_scale, max_q_len, max_prefix_q_len, out, lse)
    if type(res) is int or ops._CHECK_EVERY_CALL:
        _check(res, q.device)
    return res


def _copy(write, k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale) -> None:
    res = None
    if _binding is not None:
        res = _binding.copy(write, k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale,
                            v_scale)
    if res is None:
        validate_copy(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
        _require_cuda(k)
        if write:
            k, v = _rows_like(k), _rows_like(v)
        res = _call("copy", k.device, write, k, v, k_cache, v_cache, page_table, offsets, kv_lens,
                    k_scale, v_scale)
    if res != _native.FA_OK or ops._CHECK_EVERY_CALL:
        _check(res, k.device)


def write(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale=None, v_scale=None) -> None:
    """Write the packed rows k, v [total, heads_kv, head_dim] into the cache, in place.

    With a float8 cache each row is quantised: scale = 2^e with the smallest e >= -126 for which the
    row's largest finite magnitude is at most 448 * 2^e (1 for a row of zeros), code =
    round_e4m3(x / scale); infinities and NaN become NaN.
    """
    _copy(True, k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)


def read(k_cache, v_cache, page_table, offsets, kv_lens, total, k_scale=None, v_scale=None,
         dtype=None, out=None):
    """Read rows back: packed (k, v) [total, heads_kv, head_dim], row i of sequence b the token at
    position kv_lens[b] - (offsets[b + 1] - offsets[b]) + i.

    `total` is offsets[-1], or more (rows behind it are not written).  Rows of a float8 cache are
    dequantised and rounded to `dtype` (float16 or bfloat16, default bfloat16); others keep the
    cache's type.  `out`: a pair of tensors to fill.
    """
    if out is None:
        if dtype is None:
            dtype = torch.bfloat16 if k_cache.dtype == FP8 else k_cache.dtype
        if _binding is not None and dtype in _ROW_CODES:
            res = _binding.read_new(total, _ROW_CODES[dtype], k_cache, v_cache, page_table, offsets,
                                    kv_lens, k_scale, v_scale)
            if res is not None:
                if type(res) is int or ops._CHECK_EVERY_CALL:
                    _check(res, k_cache.device)
                return res
        try:
            total = operator.index(total)
        except TypeError:
            total = -1
        if total < 0:
            raise ValueError("total must be an integer that is not negative")
        shape = (total, k_cache.shape[1], k_cache.shape[-1])
        k = torch.empty(shape, dtype=dtype, device=k_cache.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        if k.shape[0] != total or (dtype is not None and k.dtype != dtype):
            raise ValueError("out must have `total` rows of the given dtype")
        if not (_aligned(k) and _aligned(v)) or k.is_neg() or v.is_neg():
            raise ValueError("out needs a unit inner stride and 16-byte aligned strides")
    _copy(False, k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
    return k, v


def attention_weights(q, lse, k_cache, page_table, offsets, kv_lens, weights, causal, sm_scale, k_scale=None,
                      max_q_len=None, reset_new=True) -> None:
    """Add the attention weight that each cached token gets from these rows to `weights`, in place.

    `weights` [num_pages, heads_kv, page_size] float32, a number for each (token, kv head) of the cache,
    grows by the sum of the probabilities exp(sm_scale q k - lse) of all rows and query heads that attend to
    it: `q`, `causal`, `sm_scale` and the sequences are those of the attention call that `lse` [total,
    heads_q] float32 comes from.  With `reset_new` the places of the sequences' new tokens (the last
    offsets[b + 1] - offsets[b]) start from 0, so pages need no clearing.  Rows with lse = -inf give nothing,
    whatever q holds there: a caller can leave rows out that way.  `max_q_len` as in `attention`.

    With the joint `lse` of `prefix_attention`, one call over the sequences' own tokens, and one over the
    prefixes (prefix_table, prefix_offsets, prefix_lens, causal=False, reset_new=False) give the weights of
    both.  Pages that get weight must not belong to two sequences of a call.  What a key holds shows in its
    own weight only, and what a row holds in those of the keys that it attends to.
    """
    res = None
    if _binding is not None:
        res = _binding.weights(q, lse, k_cache, page_table, offsets, kv_lens, weights, causal, sm_scale, k_scale,
                               max_q_len, bool(reset_new))
    if res is None:
        sm_scale, max_q_len = _scale(sm_scale), _max_len(max_q_len)
        validate_attention_weights(q, lse, k_cache, page_table, offsets, kv_lens, weights, k_scale, max_q_len)
        _require_cuda(q)
        if not lse.is_contiguous() or lse.is_neg():
            lse = torch.empty_like(lse, memory_format=torch.contiguous_format).copy_(lse.detach())
        res = _call("weights", q.device, _rows_like(q), lse, k_cache, page_table, offsets, kv_lens, weights,
                    bool(causal), sm_scale, k_scale, max_q_len, bool(reset_new))
    if res != _native.FA_OK or ops._CHECK_EVERY_CALL:
        _check(res, q.device)


def evict(k_cache, v_cache, weights, page_table, kv_lens, keep, recent, k_scale=None, v_scale=None,
          to_table=None):
    """Cut long sequences to `keep` tokens by the attention weight that each received; (new_lens, kept).

    `weights` [num_pages, heads_kv, page_size] float32 is what `attention_weights` accumulates.  Of a
    sequence longer than `keep` each kv head keeps its last `recent` tokens and, of the others, the
    keep - recent with the largest weights (of equal ones the earlier; NaN counts as the largest).  They
    keep their order and move to positions 0 .. keep - 1, with their scales and weights: in place, or into
    the pages of `to_table` [seqs, columns], which also receive the sequences that are not longer, and must
    not be among those of `page_table`; a row of it has to name min(kv_len, keep) places, or the call reports it
    as it does an entry outside the cache.  What lies behind the new length is left as it was.  Pages that
    receive tokens must not belong to another sequence too (a shared prefix among them).

    new_lens [seqs] int32 is min(kv_lens, keep); kept [seqs, heads_kv, keep] int32 the positions that
    stayed, -1 behind them.  Both stay on the device, and nothing waits for it.  So the launch is planned by the
    width of `page_table`: columns beyond the longest sequence cost time.
    """
    res = None
    if _binding is not None:
        res = _binding.evict(k_cache, v_cache, weights, page_table, kv_lens, keep, recent, k_scale, v_scale,
                             to_table)
    if res is None:
        keep, recent = _count(keep, "keep"), _count(recent, "recent")
        validate_evict(k_cache, v_cache, weights, page_table, kv_lens, keep, recent, k_scale, v_scale,
                       to_table)
        _require_cuda(k_cache)
        res = _call("evict", k_cache.device, k_cache, v_cache, weights, page_table, kv_lens, keep, recent,
                    k_scale, v_scale, to_table)
    if type(res) is int or ops._CHECK_EVERY_CALL:
        _check(res, k_cache.device)
    return res
