"""Paged key/value cache: writing new tokens, reading tokens back, attention over it.

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
    """Shapes, types and layout of a cache and its sequences, on tensors of any device."""
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
    if page_table.ndim != 2 or offsets.ndim != 1 or kv_lens.ndim != 1:
        raise ValueError("page_table must be [seqs, columns], offsets [seqs + 1], kv_lens [seqs]")
    seqs = page_table.shape[0]
    if offsets.shape[0] != seqs + 1 or kv_lens.shape[0] != seqs:
        raise ValueError("page_table must be [seqs, columns], offsets [seqs + 1], kv_lens [seqs]")
    if any(t.dtype != torch.int32 for t in (page_table, offsets, kv_lens)):
        raise ValueError("page_table, offsets and kv_lens must be int32")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1 or not (
            offsets.is_contiguous() and kv_lens.is_contiguous()):
        raise ValueError("offsets, kv_lens and the rows of page_table must be contiguous")
    if page_table.shape[1] * size > 1 << 30:
        raise ValueError("page_table names more than 2^30 positions a sequence")
    for t in (k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale):
        if t is not None and t.device != k_cache.device:
            raise ValueError("all tensors of a paged call must be on the same device")
        if t is not None and t.is_neg():
            raise ValueError("a cache, its scales and its sequences must not be negated views")


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
        _paged_binding.setup(*(ctypes.cast(fn, ctypes.c_void_p).value for fn in (
            lib.fa_paged_attn_sm100, lib.fa_paged_workspace_bytes, lib.fa_paged_write_sm100,
            lib.fa_paged_read_sm100)))
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


def _max_len(n):
    """An upper bound given as any kind of integer, or None."""
    if n is None:
        return None
    try:
        n = operator.index(n)
    except TypeError:
        raise ValueError(f"max_q_len must be an integer or None (got {n!r})") from None
    return min(n, 1 << 30)  # (there are no more rows)


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
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype
                                or out.device != q.device or not _aligned(out) or out.is_neg()):
            raise ValueError("out must match q in shape, dtype and device, with a unit inner stride "
                             "and 16-byte aligned strides")
        if lse is not None and (lse.shape != q.shape[:2] or lse.dtype != torch.float32
                                or lse.device != q.device or not lse.is_contiguous() or lse.is_neg()):
            raise ValueError("lse must be a contiguous float32 tensor [total, heads_q]")
        res = _call("attention", q.device, _rows_like(q), k_cache, v_cache, page_table, offsets,
                    kv_lens, bool(causal), sm_scale, k_scale, v_scale, max_q_len, out, lse)
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
