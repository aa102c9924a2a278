"""The paged cache's host side without a GPU: refusals of the Python calls and of the C ABI."""
from __future__ import annotations

import ctypes

import pytest
import torch

import flash_attention_forward as fam
import paged_ref as ref
from flash_attn_npu_b200 import _native, build

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _batch(**kw):
    return ref.Batch([2, 3], [20, 30], **kw)


def _attend(b, **kw):
    a = dict(q=b.q, k_cache=b.k_cache, v_cache=b.v_cache, page_table=b.table, offsets=b.offsets, kv_lens=b.lens,
             causal=True, sm_scale=0.1, **b.scales)
    a.update(kw)
    return fam.paged_attention(**a)


def _write(b, **kw):
    a = dict(k=b.rows[0], v=b.rows[1], k_cache=b.k_cache, v_cache=b.v_cache, page_table=b.table, offsets=b.offsets,
             kv_lens=b.lens, **b.scales)
    a.update(kw)
    return fam.paged_cache_write(**a)


@pytest.mark.parametrize("fp8", [False, True])
def test_cpu_tensors_are_refused(fp8):
    b = _batch(fp8=fp8)
    with pytest.raises(ValueError, match="CUDA"):
        _attend(b)
    with pytest.raises(ValueError, match="CUDA"):
        _write(b)
    with pytest.raises(ValueError, match="CUDA"):
        fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales)


def test_cache_and_sequence_rules():
    b, f = _batch(), _batch(fp8=True)
    bad = [
        (b, dict(k_cache=b.k_cache[0]), "same shape"),
        (b, dict(v_cache=b.v_cache[:-1]), "same shape"),
        (b, dict(v_cache=b.v_cache.half()), "float16, bfloat16 or float8"),
        (b, dict(k_cache=b.k_cache.float(), v_cache=b.v_cache.float()), "float16, bfloat16 or float8"),
        (b, dict(k_cache=b.k_cache[..., :48], v_cache=b.v_cache[..., :48]), "HEAD_DIM"),
        (b, dict(k_cache=b.k_cache[:, :, :12], v_cache=b.v_cache[:, :, :12]), "power of two"),
        (b, dict(k_cache=b.k_cache[:, :, :4], v_cache=b.v_cache[:, :, :4]), "power of two"),
        (b, dict(k_cache=b.k_cache[:0], v_cache=b.v_cache[:0]), "at least one page"),
        (b, dict(k_cache=b.k_cache.transpose(2, 3).contiguous().transpose(2, 3)), "inner stride"),
        (b, dict(v_cache=torch.zeros(*b.v_cache.shape[:3], 65).to(BF16)[..., :64]), "16-byte"),
        (b, dict(v_cache=torch.zeros(b.v_cache.numel() + 1).to(BF16)[1:].view(b.v_cache.shape)), "16-byte"),
        (b, dict(k_cache=b.k_cache[:1].expand(b.k_cache.shape)), "16-byte"),
        (b, dict(k_scale=f.k_scale, v_scale=f.v_scale), "no other"),
        (f, dict(k_scale=None), "float8_e4m3fn cache"),
        (f, dict(k_scale=None, v_scale=None), "float8_e4m3fn cache"),
        (f, dict(k_scale=f.k_scale.double()), "float32"),
        (f, dict(v_scale=f.v_scale[:, :, :8]), "num_pages, heads_kv, page_size"),
        (f, dict(v_scale=f.v_scale.transpose(1, 2).contiguous().transpose(1, 2)), "unit inner stride"),
        (b, dict(page_table=b.table.long()), "int32"),
        (b, dict(offsets=b.offsets.long()), "int32"),
        (b, dict(kv_lens=b.lens.long()), "int32"),
        (b, dict(page_table=b.table[0]), "seqs, columns"),
        (b, dict(offsets=b.offsets[:-1]), r"seqs \+ 1"),
        (b, dict(kv_lens=b.lens[:-1]), "kv_lens"),
        (b, dict(page_table=b.table.T.contiguous().T), "contiguous"),
        (b, dict(kv_lens=torch.zeros(4, dtype=torch.int32)[::2]), "contiguous"),
        (b, dict(kv_lens=b.lens.to("meta")), "same device"),
    ]
    for batch, change, text in bad:
        for call in (_attend, _write):
            with pytest.raises(ValueError, match=text):
                call(batch, **change)


def test_query_rules():
    b, f = _batch(), _batch(fp8=True)
    bad = [
        (b, dict(q=b.q[0]), "heads_q"),
        (b, dict(q=b.q[:, :3]), "multiple of heads_kv"),
        (b, dict(q=b.q[..., :32]), "head_dim"),
        (b, dict(q=b.q.half()), "cache's type"),
        (b, dict(q=b.q.float()), "float16 or bfloat16"),
        (f, dict(q=f.q.float()), "float16 or bfloat16"),
        (b, dict(q=b.q.to("meta")), "same device"),
        (b, dict(max_q_len=-1), "max_q_len"),
    ]
    for batch, change, text in bad:
        with pytest.raises(ValueError, match=text):
            _attend(batch, **change)


def test_row_rules():
    b, f = _batch(), _batch(fp8=True)
    k, v = b.rows
    bad = [
        (b, dict(k=k[:-1]), "same shape"),
        (b, dict(k=k.half()), "same shape and dtype"),
        (b, dict(k=k.half(), v=v.half()), "cache's type"),
        (f, dict(k=k.float(), v=v.float()), "float16 or bfloat16"),
        (b, dict(k=k[:, :1], v=v[:, :1]), "heads"),
        (b, dict(k=k[0], v=v[0]), "total, heads"),
    ]
    for batch, change, text in bad:
        with pytest.raises(ValueError, match=text):
            _write(batch, **change)
    for kw, text in ((dict(dtype=torch.float32), "float16 or bfloat16"), (dict(dtype=FP16), "cache's type"),
                     (dict(out=(k, v[:-1])), "same shape"), (dict(out=(k[:-1], v[:-1])), "total"),
                     (dict(out=(torch.zeros(5, 2, 65).to(BF16)[..., :64], v)), "16-byte")):
        with pytest.raises(ValueError, match=text):
            fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **kw)


def test_empty_cache():
    k, v, ks, vs = fam.paged_cache_empty(3, 16, 2, 64, FP16, "meta")
    assert k.shape == v.shape == (3, 2, 16, 64) and k.dtype == FP16 and ks is None and vs is None
    k, v, ks, vs = fam.paged_cache_empty(3, 16, 2, 64, ref.FP8, "meta")
    assert k.dtype == ref.FP8 and ks.shape == vs.shape == (3, 2, 16) and ks.dtype == torch.float32


def _args(kind, **kw):
    a = kind(struct_size=ctypes.sizeof(kind))
    c = a.cache
    c.k = c.v = 1024
    c.page_table = c.offsets = c.kv_lens = 256
    for st in (c.k_stride, c.v_stride):
        st[:] = (2 * 16 * 64, 16 * 64, 64)
    c.num_pages, c.heads_kv, c.page_size, c.head_dim, c.seqs, c.table_cols, c.table_stride = 8, 2, 16, 64, 3, 4, 4
    c.dtype = _native.FA_DTYPE_BF16
    a.total, a.dtype = 5, _native.FA_DTYPE_BF16
    if kind is _native.FaPagedAttnArgs:
        a.q = a.o = a.lse = a.workspace = 512
        a.q_stride[:] = a.o_stride[:] = (4 * 64, 64)
        a.heads_q, a.sm_scale, a.workspace_bytes = 4, 0.1, 1 << 40
    else:
        a.k = a.v = 512
        a.k_stride[:] = a.v_stride[:] = (2 * 64, 64)
    for name, x in kw.items():
        if name.startswith("c_"):
            setattr(c, name[2:], x)
        else:
            setattr(a, name, x)
    return a


def test_native_checks(native_lib):
    """Each call is refused on the host for its own reason, and a sound one stops at the device."""
    inv, mis = _native.FA_ERR_INVALID_ARG, _native.FA_ERR_MISALIGNED
    both = [
        (dict(struct_size=8), inv), (dict(c_k=0), inv), (dict(c_offsets=0), inv), (dict(c_page_table=0), inv),
        (dict(c_k=1032), mis), (dict(c_page_size=4), inv), (dict(c_page_size=24), inv), (dict(c_page_size=2048), inv),
        (dict(c_head_dim=48), _native.FA_ERR_UNSUPPORTED_HEAD_DIM), (dict(c_num_pages=0), inv),
        (dict(c_heads_kv=0), inv), (dict(c_table_cols=1 << 28), inv), (dict(c_seqs=-1), inv), (dict(total=-1), inv),
        (dict(dtype=_native.FA_DTYPE_FP32), _native.FA_ERR_UNSUPPORTED_DTYPE),
        (dict(dtype=_native.FA_DTYPE_FP16), _native.FA_ERR_UNSUPPORTED_DTYPE),
        (dict(c_dtype=7), _native.FA_ERR_UNSUPPORTED_DTYPE), (dict(c_dtype=_native.FA_DTYPE_FP8_E4M3), mis),
    ]
    attn = [(dict(heads_q=3), inv), (dict(sm_scale=float("inf")), inv), (dict(q=0), inv), (dict(workspace=0), inv),
            (dict(workspace=520), mis), (dict(q=520), mis), (dict(max_q_len=-1), inv), (dict(total=1 << 30), inv)]
    copy = [(dict(k=0), inv), (dict(v=520), mis)]
    lib = _native.load()
    for kind, fns, cases in ((_native.FaPagedAttnArgs, [lib.fa_paged_attn_sm100], both + attn),
                             (_native.FaPagedCopyArgs, [lib.fa_paged_write_sm100, lib.fa_paged_read_sm100], both + copy)):
        for fn in fns:
            for kw, want in cases:
                a = _args(kind, **kw)
                assert fn(ctypes.byref(a), None) == want, kw
            assert fn(ctypes.byref(_args(kind, total=0)), None) == _native.FA_OK
            if not torch.cuda.is_available():
                assert fn(ctypes.byref(_args(kind)), None) == _native.FA_ERR_DEVICE
    a = _args(_native.FaPagedAttnArgs, workspace=0, c_k=0, c_v=0)
    assert lib.fa_paged_workspace_bytes(ctypes.byref(a)) > 0
    a.heads_q = 3
    assert lib.fa_paged_workspace_bytes(ctypes.byref(a)) == inv
