"""Prefix attention, attention weights and eviction without a GPU: refusals of the Python calls and of the C
ABI, and the registered operators on meta and fake tensors."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_attention_forward as fam
import paged_prefix_ref as pre
import paged_ref as ref
from flash_attn_npu_b200 import _native, build, paged, torch_op  # noqa: F401  (registers the operators)

OPS = torch.ops.flash_attn_b200
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _prefix_batch(**kw):
    return pre.PrefixBatch([2, 3], [20, 30], [40, 9], [3, 2], **kw)


def _prefix(b, **kw):
    a = dict(q=b.q, k_cache=b.k_cache, v_cache=b.v_cache, prefix_table=b.prefix_table, prefix_offsets=b.prefix_offsets,
             prefix_lens=b.prefix_lens, page_table=b.table, offsets=b.offsets, kv_lens=b.lens, causal=True, sm_scale=0.1,
             **b.scales)
    a.update(kw)
    return a


def _floats(b, device=None):
    return torch.zeros(b.k_cache.shape[:3], device=device or b.k_cache.device)


def _weights(b, **kw):
    a = dict(q=b.q, lse=torch.zeros(b.q.shape[:2], device=b.q.device), k_cache=b.k_cache, page_table=b.table,
             offsets=b.offsets, kv_lens=b.lens, weights=_floats(b), causal=True, sm_scale=0.1, k_scale=b.k_scale)
    a.update(kw)
    return a


def _evict(b, **kw):
    a = dict(k_cache=b.k_cache, v_cache=b.v_cache, weights=_floats(b), page_table=b.table, kv_lens=b.lens, keep=16,
             recent=4, **b.scales)
    a.update(kw)
    return a


CALLS = {"prefix": (_prefix, fam.paged_prefix_attention, _prefix_batch),
         "weights": (_weights, fam.paged_attention_weights, lambda **kw: ref.Batch([2, 3], [20, 30], **kw)),
         "evict": (_evict, fam.paged_cache_evict, lambda **kw: ref.Batch([2, 3], [20, 30], **kw))}


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("name", list(CALLS))
def test_cpu_tensors_are_refused(name, fp8):
    args, call, batch = CALLS[name]
    with pytest.raises(ValueError, match="CUDA"):
        call(**args(batch(fp8=fp8)))


@pytest.mark.parametrize("name", list(CALLS))
def test_cache_and_sequence_rules(name):
    args, call, batch = CALLS[name]
    b, f = batch(), batch(fp8=True)
    bad = [
        (b, dict(k_cache=b.k_cache[0]), "same shape"),
        (b, dict(k_cache=b.k_cache[..., :48], v_cache=b.v_cache[..., :48]), "HEAD_DIM"),
        (b, dict(k_cache=b.k_cache[:, :, :12], v_cache=b.v_cache[:, :, :12]), "power of two"),
        (b, dict(k_cache=b.k_cache.transpose(2, 3).contiguous().transpose(2, 3)), "inner stride"),
        (b, dict(k_scale=f.k_scale, v_scale=f.v_scale), "no other"),
        (f, dict(k_scale=None, v_scale=None), "float8_e4m3fn cache"),
        (b, dict(page_table=b.table.long()), "int32"),
        (b, dict(kv_lens=b.lens.long()), "int32"),
        (b, dict(page_table=b.table[0]), "seqs, columns"),
        (b, dict(kv_lens=b.lens[:-1]), "kv_lens"),
        (b, dict(page_table=b.table.T.contiguous().T), "contiguous"),
        (b, dict(kv_lens=b.lens.to("meta")), "same device"),
    ]
    for x, change, text in bad:
        a = args(x, **change)
        if name == "weights":
            a.pop("v_cache", None), a.pop("v_scale", None)
        with pytest.raises(ValueError, match=text):
            call(**a)


def test_prefix_rules():
    b = _prefix_batch()
    for change, text in [
            (dict(prefix_table=b.prefix_table.long()), "prefix_table, prefix_offsets and prefix_lens must be int32"),
            (dict(prefix_table=b.prefix_table[0]), "prefixes, columns"),
            (dict(prefix_offsets=b.prefix_offsets[:-1]), r"prefixes \+ 1"),
            (dict(prefix_lens=b.prefix_lens[:-1]), "prefix_lens"),
            (dict(prefix_table=b.prefix_table.T.contiguous().T), "contiguous"),
            (dict(prefix_lens=b.prefix_lens.to("meta")), "same device"),
            (dict(max_prefix_q_len=-1), "max_prefix_q_len"), (dict(max_prefix_q_len="2"), "max_prefix_q_len"),
            (dict(max_q_len=-1), "max_q_len"), (dict(sm_scale=float("nan")), "sm_scale"),
            (dict(q=b.q[:, :3]), "multiple of heads_kv"), (dict(q=b.q.half()), "cache's type"),
            (dict(offsets=b.offsets[:-1]), r"seqs \+ 1")]:
        with pytest.raises(ValueError, match=text):
            fam.paged_prefix_attention(**_prefix(b, **change))


def test_weights_rules():
    b = ref.Batch([2, 3], [20, 30])
    w = _floats(b)
    for change, text in [
            (dict(lse=torch.zeros(5, 3)), "lse"), (dict(lse=torch.zeros(5, 4).double()), "lse"),
            (dict(lse=torch.zeros(5, 4, device="meta")), "lse"),
            (dict(weights=w[:, :, :8]), "weights must be float32"), (dict(weights=w.double()), "weights must be float32"),
            (dict(weights=w.transpose(1, 2).contiguous().transpose(1, 2)), "weights needs"),
            (dict(weights=torch.zeros(w.numel() + 1)[1:].view(w.shape)), "weights needs"),
            (dict(weights=w.to("meta")), "same device"), (dict(weights=w[:1].expand(w.shape)), "weights needs"),
            (dict(q=b.q[:, :3], lse=torch.zeros(5, 3)), "multiple of heads_kv"), (dict(sm_scale=float("inf")), "sm_scale"),
            (dict(max_q_len=2.5), "max_q_len")]:
        with pytest.raises(ValueError, match=text):
            fam.paged_attention_weights(**_weights(b, **change))


def test_evict_rules():
    b = ref.Batch([2, 3], [20, 30])
    t = b.table
    for change, text in [
            (dict(keep=-1, recent=-1), "keep"), (dict(keep=4, recent=5), "recent <= keep"), (dict(recent=-1), "recent"),
            (dict(keep=(1 << 30) + 1), "keep"), (dict(keep=2.0), "keep"), (dict(recent="1"), "recent"),
            (dict(weights=_floats(b).half()), "weights must be float32"),
            (dict(to_table=t.long()), "to_table"), (dict(to_table=t[:1]), "to_table"), (dict(to_table=t[0]), "to_table"),
            (dict(to_table=t.T.contiguous().T), "contiguous"), (dict(to_table=t.to("meta")), "same device")]:
        with pytest.raises(ValueError, match=text):
            fam.paged_cache_evict(**_evict(b, **change))
    with pytest.raises(ValueError, match="CUDA"):  # (NumPy integers are integers)
        fam.paged_cache_evict(**_evict(b, keep=np.int64(16), recent=np.int32(4)))


# ------------------------------------------------------------------------------ registered operators
@pytest.mark.parametrize("fp8", [False, True])
def test_fake_shapes_on_meta(fp8):
    b = _prefix_batch(fp8=fp8, dtype=FP16, device="meta")
    out, lse = OPS.paged_prefix_attention(b.q, b.k_cache, b.v_cache, *b.prefix, *b.where, True, 0.1, b.k_scale, b.v_scale)
    assert out.shape == b.q.shape and out.dtype == FP16 and lse.shape == b.q.shape[:2] and lse.dtype == torch.float32
    w = _floats(b)
    assert OPS.paged_attention_weights(b.q, lse, b.k_cache, *b.where, w, True, 0.1, b.k_scale) is None
    lens, kept = OPS.paged_cache_evict(b.k_cache, b.v_cache, w, b.table, b.lens, 16, 4, b.k_scale, b.v_scale)
    assert lens.shape == (2,) and kept.shape == (2, b.k_cache.shape[1], 16) and lens.dtype == kept.dtype == torch.int32
    with pytest.raises(ValueError, match="recent <= keep"):
        OPS.paged_cache_evict(b.k_cache, b.v_cache, w, b.table, b.lens, 16, 17, b.k_scale, b.v_scale)


def test_fake_mode():
    with FakeTensorMode():
        k, v, ks, vs = paged.empty_cache(8, 16, 2, 64, ref.FP8, "cpu")
        table, offsets, lens = (torch.zeros(s, dtype=torch.int32) for s in ((3, 2), 4, 3))
        q, w = torch.empty(5, 4, 64, dtype=BF16), torch.empty(8, 2, 16)
        out, lse = OPS.paged_prefix_attention(q, k, v, table, offsets, lens, table, offsets, lens, True, 0.1, ks, vs, 2, 3)
        assert out.shape == q.shape
        assert OPS.paged_attention_weights(q, lse, k, table, offsets, lens, w, True, 0.1, ks) is None
        assert OPS.paged_cache_evict(k, v, w, table, lens, 7, 2, ks, vs, table)[1].shape == (3, 2, 7)


# ---------------------------------------------------------------------------------------------- C ABI
def _cache(c):
    c.k = c.v = 1024
    c.page_table = c.offsets = c.kv_lens = 256
    for st in (c.k_stride, c.v_stride):
        st[:] = (2 * 16 * 64, 16 * 64, 64)
    c.num_pages, c.heads_kv, c.page_size, c.head_dim, c.seqs, c.table_cols, c.table_stride = 8, 2, 16, 64, 3, 4, 4
    c.dtype = _native.FA_DTYPE_BF16


def _native_args(kind, **kw):
    a = kind(struct_size=ctypes.sizeof(kind))
    x = a
    if kind is _native.FaPagedPrefixArgs:
        x = a.attn
        x.struct_size = ctypes.sizeof(_native.FaPagedAttnArgs)
        a.prefix_table = a.prefix_offsets = a.prefix_lens = 256
        a.prefix_stride = a.prefix_cols = 4
        a.prefixes = 2
        x.q = x.o = x.lse = 512
        x.o_stride[:] = (4 * 64, 64)
    _cache(x.cache)
    x.workspace, x.workspace_bytes = 512, 1 << 40
    if kind is _native.FaPagedEvictArgs:
        x.weights = x.new_lens = x.kept = 512
        x.keep, x.recent, x.in_place = 20, 4, 1
    else:
        x.q_stride[:] = (4 * 64, 64)
        x.total, x.dtype, x.heads_q, x.sm_scale = 5, _native.FA_DTYPE_BF16, 4, 0.1
    if kind is _native.FaPagedWeightsArgs:
        x.q = x.lse = x.weights = 512
    if kind is not _native.FaPagedPrefixArgs:
        x.weights_stride[:] = (32, 16)
    for name, v in kw.items():
        if name.startswith("c_"):
            setattr(x.cache, name[2:], v)
        elif hasattr(a, name):
            setattr(a, name, v)
        else:
            setattr(x, name, v)
    return a


def test_native_checks(native_lib):
    """Each call is refused on the host for its own reason, and a sound one stops at the device."""
    inv, mis = _native.FA_ERR_INVALID_ARG, _native.FA_ERR_MISALIGNED
    every = [(dict(struct_size=8), inv), (dict(c_k=0), inv), (dict(c_kv_lens=0), inv), (dict(c_page_table=0), inv),
             (dict(c_k=1032), mis), (dict(c_page_size=24), inv), (dict(c_head_dim=48), _native.FA_ERR_UNSUPPORTED_HEAD_DIM),
             (dict(c_num_pages=0), inv), (dict(c_table_cols=1 << 28), inv), (dict(c_seqs=-1), inv),
             (dict(c_dtype=7), _native.FA_ERR_UNSUPPORTED_DTYPE), (dict(workspace=0), inv), (dict(workspace=520), mis),
             (dict(workspace_bytes=1), inv)]
    rows = [(dict(heads_q=3), inv), (dict(sm_scale=float("inf")), inv), (dict(q=0), inv), (dict(q=520), mis),
            (dict(max_q_len=-1), inv), (dict(total=-1), inv), (dict(lse=0), inv), (dict(total=1 << 30), inv)]
    lib = _native.load()
    for kind, fn, size, cases in (
            (_native.FaPagedPrefixArgs, lib.fa_paged_prefix_sm100, lib.fa_paged_prefix_workspace_bytes,
             every + rows + [(dict(prefix_offsets=0), inv), (dict(prefix_lens=0), inv), (dict(prefix_table=0), inv),
                             (dict(prefixes=-1), inv), (dict(prefix_cols=1 << 28), inv), (dict(max_prefix_q_len=-1), inv)]),
            (_native.FaPagedWeightsArgs, lib.fa_paged_weights_sm100, lib.fa_paged_weights_workspace_bytes,
             every + rows + [(dict(weights=0), inv), (dict(weights=520), mis)]),
            (_native.FaPagedEvictArgs, lib.fa_paged_evict_sm100, lib.fa_paged_evict_workspace_bytes,
             every + [(dict(weights=0), inv), (dict(weights=520), mis), (dict(new_lens=0), inv), (dict(kept=0), inv),
                      (dict(keep=-1), inv), (dict(recent=21), inv), (dict(recent=-1), inv),
                      (dict(in_place=0, to_cols=2), inv), (dict(in_place=0, to_cols=-1), inv)])):
        for kw, want in cases:
            # (sizes are looked at before the device, and what it needs behind it)
            if "workspace_bytes" in kw and not torch.cuda.is_available() and kind is not _native.FaPagedEvictArgs:
                want = _native.FA_ERR_DEVICE
            a = _native_args(kind, **kw)
            assert fn(ctypes.byref(a), None) == want, (kind.__name__, kw)
        a = _native_args(kind, workspace=0, c_k=0)
        assert size(ctypes.byref(a)) > 0
        a = _native_args(kind, **(dict(c_seqs=0) if kind is _native.FaPagedEvictArgs else dict(total=0)))
        assert fn(ctypes.byref(a), None) == _native.FA_OK
        if not torch.cuda.is_available():
            assert fn(ctypes.byref(_native_args(kind)), None) == _native.FA_ERR_DEVICE


# ---------------------------------------------------------------------------------------------- ring slots
@pytest.mark.parametrize("name", ["fa_paged_weights.cuh", "fa_paged_tile.cuh", "fa_paged_rows.cuh"])
def test_a_slot_is_given_back_behind_its_last_reader(name):
    """Where lane 0 gives a ring's slot back for its warp, the warp has met right before: else a lane that lags
    reads what the next fill has put there.  (A race: it is looked for in the source, not by running it.)"""
    source = (build.CSRC / name).read_text()
    lines = [ln.split("//")[0].strip() for ln in source.splitlines()]
    lines = [ln for ln in lines if ln]
    gives = [i for i, ln in enumerate(lines) if "lane == 0) mbar_arrive(" in ln and "empty" in ln]
    assert gives
    for i in gives:
        before = lines[i - 1] if "tc_fence_before" not in lines[i - 1] else lines[i - 2]
        assert before == "__syncwarp();", lines[i]


def test_too_many_heads_of_sequences_are_named():
    k, v = (torch.empty(1, 65536, 8, 16, dtype=BF16, device="meta") for _ in range(2))
    w = torch.empty(1, 65536, 8, device="meta")
    table, lens = (torch.empty(s, dtype=torch.int32, device="meta") for s in ((257, 1), 257))
    with pytest.raises(ValueError, match="heads"):
        paged.validate_evict(k, v, w, table, lens, 4, 2)
    paged.validate_evict(k, v, w, table[:256], lens[:256], 4, 2)
