"""Paged calls that a user may make of the arguments as they come: rows at any address, in any layout."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_attention_forward as fam
import paged_ref as ref
from flash_attn_npu_b200 import build, ops, paged, torch_op  # noqa: F401  (registers the operators)

OPS = torch.ops.flash_attn_b200
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _off(t, by=1):
    """The same values, contiguous, `by` elements behind an aligned address."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    out = flat[by:by + t.numel()].view(t.shape)
    out.copy_(t)
    return out


def _permuted(t, by=0):
    """The same values with the heads outside the tokens, `by` elements behind an aligned address."""
    return _off(t.transpose(0, 1).contiguous(), by).transpose(0, 1)


def _layouts(t):
    wide = torch.empty(*t.shape[:2], t.shape[2] + 3, dtype=t.dtype, device=t.device)[..., 1:1 + t.shape[2]]
    return {"contiguous, odd address": _off(t), "permuted": _permuted(t), "permuted, odd address": _permuted(t, 3),
            "odd strides": wide.copy_(t), "shared by the heads": t[:, :1].expand(t.shape)}


def test_rows_of_any_layout_become_aligned():
    t = torch.randn(5, 4, 64).to(BF16)
    for name, x in _layouts(t).items():
        y = paged._rows_like(x)
        assert paged._aligned(y), name
        assert torch.equal(x, y), name
        assert y.stride() == paged.empty_rows(x).stride(), name
    assert paged._rows_like(t) is t
    assert paged._rows_like(_permuted(t, 3)).stride() == _permuted(t).stride()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_rows_of_any_layout(fp8, cuda_device):
    b = ref.Batch([1, 30, 140], [500, 77, 300], heads_q=4, heads_kv=2, head_dim=64, fp8=fp8, device=cuda_device, garbage=0.0)
    given = {n: getattr(b, n).clone() for n in ("k_cache", "v_cache") + (("k_scale", "v_scale") if fp8 else ())}
    for name, q in _layouts(b.q).items():
        want, want_lse = fam.paged_attention(q.contiguous().clone(), b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales,
                                             return_lse=True)
        out, lse = fam.paged_attention(q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), name
        assert out.stride() == paged.empty_rows(q).stride(), name
    for name in _layouts(b.rows[0]):
        held = []
        for rows in (_layouts, lambda t: {name: _layouts(t)[name].contiguous().clone()}):
            for n, x in given.items():
                getattr(b, n).copy_(x)
            k, v = (rows(x)[name] for x in b.rows)
            fam.paged_cache_write(k, v, b.k_cache, b.v_cache, *b.where, **b.scales)
            held.append([getattr(b, n).view(torch.uint8).clone() for n in given])
        for x, y in zip(*held):
            assert torch.equal(x, y), name
    ops.check_device_status(cuda_device)


@pytest.mark.gpu
def test_registered_operator_in_any_layout(cuda_device):
    """The traced call foresees the output's layout whatever the address is."""
    b = ref.Batch([1, 30], [50, 77], heads_q=4, heads_kv=2, head_dim=64, device=cuda_device, garbage=0.0)
    for q in _layouts(b.q).values():
        torch.library.opcheck(OPS.paged_attention, (q, b.k_cache, b.v_cache, *b.where, True, 0.1),
                              test_utils=("test_schema", "test_faketensor"))


# ------------------------------------------------------------------------------ refusals and their reasons
def _attend(b, **kw):
    a = dict(q=b.q, k_cache=b.k_cache, v_cache=b.v_cache, page_table=b.table, offsets=b.offsets, kv_lens=b.lens,
             causal=True, sm_scale=0.1, **b.scales)
    a.update(kw)
    return fam.paged_attention(**a)


BAD = [(dict(sm_scale=float("inf")), "sm_scale"), (dict(sm_scale=float("nan")), "sm_scale"), (dict(sm_scale=1e300), "sm_scale"),
       (dict(sm_scale=None), "sm_scale"), (dict(max_q_len=2.0), "max_q_len"), (dict(max_q_len="2"), "max_q_len"),
       (dict(max_q_len=np.int64(-1)), "max_q_len")]


def test_scales_and_lengths_are_refused_for_what_they_are():
    b = ref.Batch([2, 3], [20, 30])
    for change, text in BAD:
        with pytest.raises(ValueError, match=text):
            _attend(b, **change)


def test_sizes_beyond_the_library():
    b = ref.Batch([2, 3], [20, 30], device="meta")
    shape = list(b.k_cache.shape)
    for at, n, text in ((0, (1 << 30) + 1, "pages"), (1, 65537, "heads")):
        many = [*shape[:at], n, *shape[at + 1:]]
        k = torch.empty_strided(many, b.k_cache.stride(), dtype=BF16, device="meta")
        with pytest.raises(ValueError, match=text):
            paged.validate_cache(k, k, *b.where, None, None)
    k = torch.empty_strided(shape, (1 << 38, *b.k_cache.stride()[1:]), dtype=BF16, device="meta")
    with pytest.raises(ValueError, match="2\\^38"):
        paged.validate_cache(k, k, *b.where, None, None)


@pytest.mark.gpu
def test_reasons_and_integers_on_the_device(cuda_device):
    b = ref.Batch([1, 30], [50, 77], heads_q=4, heads_kv=2, head_dim=64, device=cuda_device)
    want = _attend(b)
    for n in (30, np.int64(30), np.int32(30), torch.tensor(30), 1 << 70):
        assert torch.equal(_attend(b, max_q_len=n), want)
    for scale in (np.float32(0.1), torch.tensor(0.1)):
        assert torch.allclose(_attend(b, sm_scale=scale).float(), want.float())
    for change, text in BAD:
        with pytest.raises(ValueError, match=text):
            _attend(b, **change)
    with FakeTensorMode() as mode, pytest.raises(ValueError, match="subclass"):
        fake = [mode.from_tensor(x) for x in (b.q, b.k_cache, b.v_cache, *b.where)]
        paged.attention(*fake, True, 0.1)


# ------------------------------------------------------------------------------ negated views
def test_negated_views_are_copied_or_refused():
    b = ref.Batch([2, 3], [20, 30])
    x = paged._rows_like(torch._neg_view(b.q))
    assert not x.is_neg() and torch.equal(x, -b.q)
    for name in ("k_cache", "v_cache"):
        with pytest.raises(ValueError, match="negated"):
            _attend(b, **{name: torch._neg_view(getattr(b, name))})


@pytest.mark.gpu
def test_negated_views(cuda_device):
    """Their memory holds the values with the other sign."""
    b = ref.Batch([1, 30], [50, 77], heads_q=4, heads_kv=2, head_dim=64, device=cuda_device, garbage=0.0)
    want = _attend(b)
    assert torch.equal(_attend(b, q=torch._neg_view(-b.q)), want)
    with pytest.raises(ValueError, match="out"):
        _attend(b, out=torch._neg_view(torch.empty_like(b.q)))
    with pytest.raises(ValueError, match="negated"):
        _attend(b, v_cache=torch._neg_view(b.v_cache))
    k, v = b.rows
    fam.paged_cache_write(k, v, b.k_cache, b.v_cache, *b.where)
    held = b.k_cache.clone(), b.v_cache.clone()
    fam.paged_cache_write(torch._neg_view(-k), torch._neg_view(-v), b.k_cache, b.v_cache, *b.where)
    assert torch.equal(held[0], b.k_cache) and torch.equal(held[1], b.v_cache)
    ops.check_device_status(cuda_device)


# ------------------------------------------------------------------------------ what autograd sees
@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_tensors_written_in_place_have_a_new_version(fp8, cuda_device):
    b = ref.Batch([1, 30], [50, 77], heads_q=4, heads_kv=2, head_dim=64, fp8=fp8, device=cuda_device, garbage=0.0)
    held = [b.k_cache, b.v_cache] + ([b.k_scale, b.v_scale] if fp8 else [])
    out, lse = torch.empty_like(b.q), torch.empty(b.q.shape[:2], device=cuda_device)
    back = [torch.empty_like(x) for x in b.rows]

    def versions(ts):
        return [t._version for t in ts]

    before = versions(held + [out, lse] + back)
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where, **b.scales)
    _attend(b, out=out, lse=lse)
    fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales, out=tuple(back))
    assert all(x > y for x, y in zip(versions(held + [out, lse] + back), before))
    now = versions([b.q, b.table, b.offsets, b.lens, *b.rows] + held)
    _attend(b)
    fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales)
    assert versions([b.q, b.table, b.offsets, b.lens, *b.rows] + held) == now


@pytest.mark.gpu
def test_backward_over_a_cache_written_meanwhile_is_refused(cuda_device):
    b = ref.Batch([3], [20], heads_kv=2, head_dim=64, device=cuda_device, garbage=0.0)
    w = torch.ones((), device=cuda_device, requires_grad=True)
    loss = (w * b.k_cache).sum()
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_inference_tensors_may_be_written(cuda_device):
    with torch.inference_mode():
        b = ref.Batch([3], [20], heads_kv=2, head_dim=64, device=cuda_device, garbage=0.0)
        fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where)
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where)
    out = torch.zeros_like(b.q)
    _attend(b, out=out)
    assert (out != 0).any()


# ------------------------------------------------------------------------------ caches and sequences as they come
def _cut(b, how):
    """The batch's cache, its scales too, as views of larger tensors."""
    for names in (("k_cache", "v_cache"), ("k_scale", "v_scale")):
        k, v = (getattr(b, n) for n in names)
        if k is None:
            continue
        raw = [x.view(torch.uint8) if x.dtype == ref.FP8 else x for x in (k, v)]
        if how == "joint":            # [pages, K and V, heads, ..]
            both = torch.stack(raw, 1)
            cut = both[:, 0], both[:, 1]
        elif how == "pages inside":   # [heads, pages, ..]
            cut = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in raw]
        else:                         # some of the heads and pages of a larger cache
            cut = []
            for x in raw:
                big = torch.zeros(x.shape[0] + 4, x.shape[1] + 3, *x.shape[2:], dtype=x.dtype, device=x.device)
                cut.append(big[3:-1, 1:-2].copy_(x))
        for n, x in zip(names, cut):
            setattr(b, n, x.view(ref.FP8) if k.dtype == ref.FP8 else x)
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("how", ["joint", "pages inside", "some"])
@pytest.mark.parametrize("counts", [[1, 2, 1], [30, 140, 1]])
def test_caches_cut_from_larger_tensors(counts, how, fp8, cuda_device):
    a, b = (ref.Batch(counts, [500, 177, 300], heads_q=8, heads_kv=2, head_dim=64, page=32, fp8=fp8, device=cuda_device,
                      garbage=0.0) for _ in range(2))
    _cut(b, how)
    most = max(counts)
    assert torch.equal(_attend(a, max_q_len=most), _attend(b, max_q_len=most))
    for x in (a, b):
        fam.paged_cache_write(*x.rows, x.k_cache, x.v_cache, *x.where, **x.scales)
    for n in ("k_cache", "v_cache") + (("k_scale", "v_scale") if fp8 else ()):
        assert torch.equal(getattr(a, n).float(), getattr(b, n).float()), n
    for x, y in zip(*(fam.paged_cache_read(z.k_cache, z.v_cache, *z.where, z.total, **z.scales) for z in (a, b))):
        assert torch.equal(x, y)
    ops.check_device_status(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("count", [1, 50])
def test_sequences_that_share_a_row_of_the_table(count, fp8, cuda_device):
    """One row of the table for all, expanded: the same tokens seen at different lengths."""
    b = ref.Batch([count] * 3, [300] * 3, heads_q=8, heads_kv=2, head_dim=64, fp8=fp8, device=cuda_device, garbage=0.0)
    b.lens = torch.tensor([300, 211, 64], dtype=torch.int32, device=cuda_device)
    b.table = b.table[:1].expand(3, b.table.shape[1])
    assert b.table.stride(0) == 0
    out = _attend(b, max_q_len=count)
    b.table = b.table.contiguous()
    assert torch.equal(out, _attend(b, max_q_len=count))
    want, _, tol, _ = ref.attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales, max_q_len=count)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("counts", [[1, 2], [30, 140]])
def test_rows_before_the_first_sequence_are_padding(counts, fp8, cuda_device):
    b = ref.Batch(counts, [500, 177], heads_q=4, heads_kv=2, head_dim=64, fp8=fp8, device=cuda_device, garbage=0.0, pad=7)
    n, most = int(b.offsets[-1]), max(counts)
    want = _attend(b, max_q_len=most)
    caches = [b.k_cache, b.v_cache] + ([b.k_scale, b.v_scale] if fp8 else [])
    held = [x.clone() for x in caches]
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where, **b.scales)
    read = fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales)
    written = [x.clone() for x in caches]
    for x, y in zip(caches, held):
        x.copy_(y)
    b.offsets += 5
    q = torch.full_like(b.q, 7.0)
    q[5:5 + n] = b.q[:n]
    out, lse = torch.full_like(b.q, 7.0), torch.full(b.q.shape[:2], 7.0, device=cuda_device)
    _attend(b, q=q, out=out, lse=lse, max_q_len=most)
    assert torch.equal(out[5:5 + n], want[:n])
    for x in (out, lse):
        assert (x[:5] == 7).all() and (x[5 + n:] == 7).all()
    rows = [torch.full_like(x, 7.0) for x in b.rows]
    for x, y in zip(rows, b.rows):
        x[5:5 + n] = y[:n]
    fam.paged_cache_write(*rows, b.k_cache, b.v_cache, *b.where, **b.scales)
    for x, y in zip(caches, written):
        assert torch.equal(x.float(), y.float())
    back = tuple(torch.full_like(x, 7.0) for x in b.rows)
    fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales, out=back)
    for x, y in zip(back, read):
        assert torch.equal(x[5:5 + n], y[:n]) and (x[:5] == 7).all() and (x[5 + n:] == 7).all()
    ops.check_device_status(cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_a_table_without_columns(fp8, cuda_device):
    for counts in ([1, 1], [40, 2]):
        b = ref.Batch(counts, [40, 2], heads_q=4, heads_kv=2, head_dim=64, fp8=fp8, device=cuda_device)
        b.table, b.lens = b.table[:, :0], torch.zeros_like(b.lens)
        out, lse = _attend(b, return_lse=True, max_q_len=max(counts))
        assert (out == 0).all() and torch.isneginf(lse).all()
    ops.check_device_status(cuda_device)


@pytest.mark.gpu
def test_the_output_may_be_the_queries(cuda_device):
    for counts in ([1, 2], [30, 300]):
        b = ref.Batch(counts, [5000, 777], heads_q=8, heads_kv=2, head_dim=128, device=cuda_device)
        want = _attend(b, max_q_len=max(counts))
        q = b.q.clone()
        assert torch.equal(_attend(b, q=q, out=q, max_q_len=max(counts)), want)


def test_totals_that_are_none():
    b = ref.Batch([2, 3], [20, 30])
    for total, text in ((-1, "total"), (2.5, "total"), ("5", "total")):
        with pytest.raises(ValueError, match=text):
            fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, total)
