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
mix them.  Packed rows behind offsets[-1] are padding: they are not read, and outputs there are
left as they were.  Pages behind a sequence's length may hold anything, NaN included.

A float8 cache holds code = round_e4m3(x / scale) with one power of two per (token, kv head); any
positive scale can be read.  page_size is a power of two, 8 .. 1024.  Two sequences may share pages (a
common prefix), but a call to `write` must not be given the same place twice: which of the rows
stays there is open.

`page_table`, `kv_lens` and `offsets` are device data, which a launch does not wait for.  Entries outside
the cache or the table are never followed: the call reports them through the device status word
(`ops.check_device_status` raises), and the results of that sequence are undefined.
"""
from __future__ import annotations

import ctypes
import struct

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
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not _aligned(t):
            raise ValueError(f"{name} needs a unit inner stride and 16-byte aligned strides")
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
    for t in (v_cache, page_table, offsets, kv_lens, k_scale, v_scale):
        if t is not None and t.device != k_cache.device:
            raise ValueError("all tensors of a paged call must be on the same device")


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


def _aligned(t) -> bool:
    """Unit inner stride, and 16-byte strides and address (of a tensor that has one)."""
    eb = t.element_size()
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return False
    if any(t.shape[d] > 1 and (t.stride(d) <= 0 or (t.stride(d) * eb) % 16)
           for d in range(t.ndim - 1)):
        return False
    return t.device.type == "meta" or t.data_ptr() % 16 == 0


def _strides(t) -> tuple:
    """Strides of the outer dimensions, a contiguous one where a dimension of size 1 has any."""
    out, inner = [], t.shape[-1]
    for d in range(t.ndim - 2, -1, -1):
        st = t.stride(d) if t.shape[d] > 1 else inner
        out.append(st)
        inner = max(inner, st * t.shape[d])
    return tuple(reversed(out))


def _require_cuda(t) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"paged calls take CUDA tensors on an sm_100 device (got {t.device})")


# ------------------------------------------------------------------------------------ launching
# A call's argument block has its addresses first (PREFIX) and its layout behind them.  The layout
# part of a call that was validated and launched once is kept under the call's shapes, strides,
# types and options, so a call of the same layout only fills in its addresses: the full checks cost
# several times what a decoding step's kernel takes.  Nothing is kept by address.
_FAST: dict = {}
_FAST_LIMIT = 256
_ATTN_PTRS = struct.Struct("@12Q")  # q, o, lse, workspace, status, k, v, scales, table, offsets, lens
_COPY_PTRS = struct.Struct("@10Q")  # k, v, status, k, v, scales, table, offsets, lens
_PTRS_AT = 8                        # behind struct_size


def _remember(key, value) -> None:
    if len(_FAST) >= _FAST_LIMIT:
        _FAST.pop(next(iter(_FAST)))
    _FAST[key] = value


def _fill_cache(c, k_cache, v_cache, page_table, k_scale, v_scale) -> None:
    for name, t in (("k_stride", k_cache), ("v_stride", v_cache)):
        getattr(c, name)[:] = _strides(t)
    if k_scale is not None:
        for name, t in (("k_scale_stride", k_scale), ("v_scale_stride", v_scale)):
            getattr(c, name)[:] = _strides(t)
    c.num_pages, c.heads_kv, c.page_size, c.head_dim = k_cache.shape
    c.seqs, c.table_cols = page_table.shape
    c.table_stride = page_table.stride(0) if page_table.shape[0] > 1 else page_table.shape[1]
    c.dtype = _CACHE_CODES[k_cache.dtype]


def _status_of(device):
    """The device's status word, or None in a capture that comes before its first launch (an
    allocation there would belong to the graph's private pool)."""
    if (ops._device_index(device) in ops._STATUS_WORDS
            or not torch.cuda.is_current_stream_capturing()):
        return ops.device_status_word(device)
    return None


def _launch(fn, block, index) -> None:
    """Launch on the current stream of device `index`, whatever device is current."""
    buf = (ctypes.c_char * len(block)).from_buffer(block)
    if torch._C._cuda_getDevice() == index:
        rc = fn(buf, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(buf, torch._C._cuda_getCurrentRawStream(index))
    if rc != _native.FA_OK:
        exc = _native.NativeError(rc, _native.status_string(rc))
        if rc in (_native.FA_ERR_UNSUPPORTED_HEAD_DIM, _native.FA_ERR_UNSUPPORTED_DTYPE,
                  _native.FA_ERR_INVALID_ARG, _native.FA_ERR_MISALIGNED):
            raise ValueError(str(exc)) from None
        raise exc
    if ops._CHECK_EVERY_CALL:
        ops.check_device_status(torch.device("cuda", index))


def _layout(*tensors):
    return tuple((t.shape, t.stride(), t.dtype, t.device) if t is not None else None
                 for t in tensors)


def _rows_like(t):
    """`t`, or a contiguous copy where its rows are not 16-byte aligned."""
    return t if _aligned(t) else t.contiguous()


def attention(q, k_cache, v_cache, page_table, offsets, kv_lens, causal, sm_scale, k_scale=None,
              v_scale=None, max_q_len=None, out=None, lse=None):
    """Attention of the packed queries q [total, heads_q, head_dim] over the cache; (out, lse).

    Query head h reads kv head h // (heads_q // heads_kv).  Causal: a token attends to positions up
    to its own; else to its whole sequence.  `out` is like q, `lse` [total, heads_q] float32 the
    natural-log logsumexp; a row with no key to attend to gets 0 and -inf.  `max_q_len`: an upper
    bound of a sequence's new tokens that the kernel choice goes by (default: total).  `out` and
    `lse` may be given; rows that belong to no sequence are not written.
    """
    key = ("attention", _layout(q, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale),
           bool(causal), float(sm_scale), max_q_len)
    ent = _FAST.get(key)
    if ent is None:
        validate_attention(q, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale,
                           max_q_len)
        _require_cuda(q)
    q = _rows_like(q)
    if out is None:
        out = torch.empty_like(q)
        if not _aligned(out):
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not _aligned(out):
        raise ValueError("out must match q in shape, dtype and device, with a unit inner stride and "
                         "16-byte aligned strides")
    if lse is None:
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    elif (lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.device != q.device
          or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous float32 tensor [total, heads_q]")
    if q.shape[0] == 0 or page_table.shape[0] == 0:
        return out, lse
    if ent is None:
        args = _native.FaPagedAttnArgs(struct_size=ctypes.sizeof(_native.FaPagedAttnArgs))
        _fill_cache(args.cache, k_cache, v_cache, page_table, k_scale, v_scale)
        args.total, args.heads_q = q.shape[:2]
        args.max_q_len = 0 if max_q_len is None else int(max_q_len)
        args.dtype, args.causal = _ROW_CODES[q.dtype], int(bool(causal))
        args.sm_scale = float(sm_scale)
        ent = (args, ops._device_index(q.device))
    args, index = ent
    block = bytearray(args)
    _STRIDES.pack_into(block, _Q_STRIDE_AT, *_strides(q), *_strides(out))
    return _attention_launch(key, args, index, block, q, k_cache, v_cache, page_table, offsets,
                             kv_lens, k_scale, v_scale, out, lse)


_STRIDES = struct.Struct("@4q")
_Q_STRIDE_AT = _native.FaPagedAttnArgs.q_stride.offset
_COPY_STRIDE_AT = _native.FaPagedCopyArgs.k_stride.offset


def _attention_launch(key, args, index, block, q, k_cache, v_cache, page_table, offsets, kv_lens,
                      k_scale, v_scale, out, lse):
    lib = _native.load()
    if args.workspace_bytes == 0:
        with torch.cuda.device(index):
            need = lib.fa_paged_workspace_bytes(ctypes.byref(args))
        if need < 0:
            raise ValueError(_native.status_string(need))
        args.workspace_bytes = need
        block[_WS_AT:_WS_AT + 8] = struct.pack("@q", need)
    workspace = torch.empty(args.workspace_bytes, dtype=torch.uint8, device=q.device)
    status = _status_of(q.device)
    _ATTN_PTRS.pack_into(
        block, _PTRS_AT, q.data_ptr(), out.data_ptr(), lse.data_ptr(), workspace.data_ptr(),
        status.data_ptr() if status is not None else 0, k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr() if k_scale is not None else 0,
        v_scale.data_ptr() if v_scale is not None else 0, page_table.data_ptr(),
        offsets.data_ptr(), kv_lens.data_ptr())
    _launch(lib.fa_paged_attn_sm100, block, index)
    if key not in _FAST:
        _remember(key, (args, index))
    return out, lse


_WS_AT = _native.FaPagedAttnArgs.workspace_bytes.offset


def _copy(fn_name, k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale, key):
    if k.shape[0] == 0 or page_table.shape[0] == 0:
        return
    ent = _FAST.get(key)
    if ent is None:
        args = _native.FaPagedCopyArgs(struct_size=ctypes.sizeof(_native.FaPagedCopyArgs))
        _fill_cache(args.cache, k_cache, v_cache, page_table, k_scale, v_scale)
        args.total, args.dtype = k.shape[0], _ROW_CODES[k.dtype]
        ent = (args, ops._device_index(k.device))
    args, index = ent
    block = bytearray(args)
    _STRIDES.pack_into(block, _COPY_STRIDE_AT, *_strides(k), *_strides(v))
    status = _status_of(k.device)
    _COPY_PTRS.pack_into(
        block, _PTRS_AT, k.data_ptr(), v.data_ptr(),
        status.data_ptr() if status is not None else 0, k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr() if k_scale is not None else 0,
        v_scale.data_ptr() if v_scale is not None else 0, page_table.data_ptr(),
        offsets.data_ptr(), kv_lens.data_ptr())
    _launch(getattr(_native.load(), fn_name), block, index)
    if key not in _FAST:
        _remember(key, ent)


def write(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale=None, v_scale=None) -> None:
    """Write the packed rows k, v [total, heads_kv, head_dim] into the cache, in place.

    With a float8 cache each row is quantised: scale = 2^e with the smallest e >= -126 for which the
    row's largest finite magnitude is at most 448 * 2^e (1 for a row of zeros), code =
    round_e4m3(x / scale); infinities and NaN become NaN.
    """
    key = ("write", _layout(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale))
    if key not in _FAST:
        validate_copy(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
        _require_cuda(k)
    _copy("fa_paged_write_sm100", _rows_like(k), _rows_like(v), k_cache, v_cache, page_table,
          offsets, kv_lens, k_scale, v_scale, key)


def read(k_cache, v_cache, page_table, offsets, kv_lens, total, k_scale=None, v_scale=None,
         dtype=None, out=None):
    """Read rows back: packed (k, v) [total, heads_kv, head_dim], row i of sequence b the token at
    position kv_lens[b] - (offsets[b + 1] - offsets[b]) + i.

    `total` is offsets[-1], or more (rows behind it are not written).  Rows of a float8 cache are
    dequantised and rounded to `dtype` (float16 or bfloat16, default bfloat16); others keep the cache's
    type.  `out`: a pair of tensors to fill.
    """
    if out is None:
        if dtype is None:
            dtype = torch.bfloat16 if k_cache.dtype == FP8 else k_cache.dtype
        shape = (int(total), k_cache.shape[1], k_cache.shape[-1])
        k, v = (torch.empty(shape, dtype=dtype, device=k_cache.device) for _ in range(2))
    else:
        k, v = out
        if k.shape[0] != total or (dtype is not None and k.dtype != dtype):
            raise ValueError("out must have `total` rows of the given dtype")
        if not (_aligned(k) and _aligned(v)):
            raise ValueError("out needs a unit inner stride and 16-byte aligned strides")
    key = ("read", _layout(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale))
    if key not in _FAST:
        validate_copy(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
        _require_cuda(k)
    _copy("fa_paged_read_sm100", k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale,
          v_scale, key)
    return k, v
