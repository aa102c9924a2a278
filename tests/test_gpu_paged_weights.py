"""The attention weights of cached tokens against their 64-bit form (B200)."""
from __future__ import annotations

import pytest
import torch

import flash_attention_forward as fam
import paged_prefix_ref as pre
import paged_ref as ref
import paged_weights_ref as ref_w
from flash_attn_npu_b200 import build, ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _check(b, causal=True, scale=None, max_q_len=None, reset_new=True, lse=None):
    scale = b.q.shape[-1] ** -0.5 if scale is None else scale
    if lse is None:
        lse = ref_w.logsumexps(b, causal, scale)
    g = torch.Generator().manual_seed(11)
    old = torch.rand(b.k_cache.shape[:3], generator=g).to(b.q.device)
    w = old.clone()
    fam.paged_attention_weights(b.q, lse, b.k_cache, *b.where, w, causal, scale, k_scale=b.k_scale,
                                max_q_len=max_q_len, reset_new=reset_new)
    ops.check_device_status(b.q.device)
    want, tol = ref_w.weights(b, lse, old, causal, scale, reset_new)
    over = (w.double() - want).abs() - tol
    assert not (over > 0).any() and not torch.isnan(over).any(), over.max().item()
    assert torch.equal(w[tol == 0], old[tol == 0])  # places of no sequence
    return w


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128, 256])
def test_decoding(head_dim, dtype, fp8, cuda_device):
    lens = [1, 7, 8, 127, 128, 129, 255, 256, 257, 600, 1, 1000]
    b = ref.Batch([1] * len(lens), lens, heads_q=8, heads_kv=2, head_dim=head_dim, page=16, dtype=dtype, fp8=fp8,
                  device=cuda_device, seed=head_dim)
    _check(b, max_q_len=1)
    _check(b)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128, 256])
def test_chunks(head_dim, fp8, causal, cuda_device):
    counts = [5, 0, 1, 33, 64, 130, 300]
    lens = [5, 40, 1, 200, 64, 513, 900]
    b = ref.Batch(counts, lens, heads_q=6, heads_kv=2, head_dim=head_dim, page=32, fp8=fp8,
                  dtype=FP16 if head_dim in (32, 128) else BF16, device=cuda_device, seed=1)
    _check(b, causal)
    _check(b, causal, max_q_len=1, reset_new=False)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("fp8", [False, True])
def test_page_sizes(page, fp8, cuda_device):
    _check(ref.Batch([1, 20, 3], [page, 2 * page + 5, 3 * page - 1] if page > 8 else [8, 21, 23], head_dim=128,
                     page=page, fp8=fp8, device=cuda_device, seed=2))


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (5, 5), (7, 1), (16, 1), (17, 1), (64, 2), (40, 1), (129, 1), (300, 1)])
@pytest.mark.parametrize("head_dim,fp8", [(64, False), (128, True), (256, True), (256, False)])
def test_head_groups(heads, head_dim, fp8, cuda_device):
    """Groups that leave rows of a query tile over, and that need several tiles."""
    b = ref.Batch([1, 9, 2], [300, 77, 2], heads_q=heads[0], heads_kv=heads[1], head_dim=head_dim, fp8=fp8,
                  device=cuda_device, seed=3)
    _check(b)
    _check(b, max_q_len=1)


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_without_keys(fp8, cuda_device):
    """Empty sequences, chunks longer than what the cache holds, sequences without new tokens."""
    b = ref.Batch([1, 200, 0, 40, 3], [0, 0, 100, 10, 3], head_dim=64, fp8=fp8, device=cuda_device, seed=4)
    _check(b, True)
    _check(b, False)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("counts,lens", [([2000], [2000]), ([700, 1], [700, 9000]), ([300], [20000]), ([1100, 900], [1200, 905])])
def test_items_shared_among_ctas(counts, lens, fp8, cuda_device):
    b = ref.Batch(counts, lens, heads_q=4, heads_kv=1, head_dim=64, page=64, fp8=fp8, device=cuda_device, seed=5)
    first = _check(b)
    assert all(torch.equal(_check(b), first) for _ in range(2))
    _check(b, False)


def test_many_sequences(cuda_device):
    counts = [(i * 7) % 5 for i in range(300)]
    lens = [c + (i * 13) % 90 for i, c in enumerate(counts)]
    _check(ref.Batch(counts, lens, heads_q=4, heads_kv=2, head_dim=64, page=8, device=cuda_device, seed=6), max_q_len=4)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_scales(scale, cuda_device):
    _check(ref.Batch([1, 30], [77, 40], head_dim=64, device=cuda_device, seed=7), scale=scale)


def test_layouts_and_padding(cuda_device):
    b = ref.Batch([3, 20], [200, 300], head_dim=64, layout="rows", device=cuda_device, seed=8, pad=5)
    b.offsets += 2
    b.q[:2] = float("nan")
    b.q[25:] = float("nan")
    lse = ref_w.logsumexps(b, True, 0.125)
    lse[:2] = lse[25:] = float("nan")
    _check(b, lse=lse, scale=0.125)
    odd = torch.empty(b.q.shape[0], b.q.shape[1], 65, dtype=b.q.dtype, device=cuda_device)[..., 1:]
    odd.copy_(b.q)
    b.q = odd  # rows at odd addresses are copied first
    _check(b, lse=lse.T.contiguous().T, scale=0.125)


def test_a_bad_key_or_row_shows_where_it_belongs(cuda_device):
    b = ref.Batch([4], [200], heads_q=2, heads_kv=1, head_dim=64, page=64, device=cuda_device, seed=9)
    lse = ref_w.logsumexps(b, True, 0.125)
    w, z = torch.zeros(b.k_cache.shape[:3], device=cuda_device), torch.zeros(b.k_cache.shape[:3], device=cuda_device)
    args = (b.k_cache, *b.where)
    fam.paged_attention_weights(b.q, lse, *args, w, True, 0.125)
    b.k_cache[b.table[0, 1], 0, 5] = float("nan")  # position 69
    b.q[2, 0, 3] = float("inf")                    # token 198 gives to 0 .. 198
    fam.paged_attention_weights(b.q, lse, *args, z, True, 0.125)
    flat = z[b.table[0].long(), 0].flatten()
    assert torch.isnan(flat[69])
    assert flat[199] == w[b.table[0].long(), 0].flatten()[199]


def test_prefix_and_own_tokens(cuda_device):
    """With the joint logsumexp the weights of prefix and own tokens add up to the number of rows."""
    x = pre.PrefixBatch([1, 6, 40, 1], [50, 6, 300, 1], [700], [48], heads_q=8, heads_kv=2, head_dim=64,
                        device=cuda_device, seed=10)
    lse = fam.paged_prefix_attention(x.q, x.k_cache, x.v_cache, *x.prefix, *x.where, True, 0.125, return_lse=True)[1]
    w = torch.zeros(x.k_cache.shape[:3], device=cuda_device)
    fam.paged_attention_weights(x.q, lse, x.k_cache, *x.where, w, True, 0.125)
    fam.paged_attention_weights(x.q, lse, x.k_cache, *x.prefix, w, False, 0.125, reset_new=False)
    torch.testing.assert_close(w.sum((0, 2)), torch.full((2,), 48 * 4.0, device=cuda_device), atol=0, rtol=1e-4)


def test_captured_step(cuda_device):
    b = ref.Batch([1] * 9 + [70], [100 * i + 1 for i in range(9)] + [90], heads_q=8, heads_kv=2, head_dim=128,
                  device=cuda_device, seed=12)
    lse = ref_w.logsumexps(b, True, 0.1)
    w = torch.zeros(b.k_cache.shape[:3], device=cuda_device)
    args = (b.q, lse, b.k_cache, *b.where)
    fam.paged_attention_weights(*args, w, True, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fam.paged_attention_weights(*args, w, True, 0.1)
    b.lens -= 1
    b.lens.clamp_(min=1)
    z = w.clone()
    graph.replay()
    fam.paged_attention_weights(*args, z, True, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(w, z)


def test_pages_that_are_none_are_reported(cuda_device):
    b = ref.Batch([1, 40], [200, 300], head_dim=64, device=cuda_device, seed=4)
    lse = ref_w.logsumexps(b, True, 0.1)
    w = torch.zeros(b.k_cache.shape[:3], device=cuda_device)
    b.table = b.table.clone()
    free = [i for i in range(w.shape[0]) if i not in set(b.table.flatten().tolist())]
    b.table[0, 2], b.table[1, 3] = 10 ** 6, -3
    fam.paged_attention_weights(b.q, lse, b.k_cache, *b.where, w, True, 0.1)
    with pytest.raises(RuntimeError, match="page"):
        ops.check_device_status(cuda_device)
    ops.check_device_status(cuda_device)
    assert (w[free] == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lse", [float("-inf"), 200.0])
def test_rows_that_give_nothing(lse, fp8, cuda_device):
    """Not even the smallest number: equal weights stay equal.  (exp(-200 + |s|), |s| < 64, is below 2^-150.)"""
    b = ref.Batch([130, 1, 70], [500, 300, 70], heads_q=4, heads_kv=2, head_dim=64, page=32, fp8=fp8, dtype=BF16,
                  device=cuda_device, seed=8)
    b.q.div_(16)
    w = torch.zeros(b.k_cache.shape[:3], device=cuda_device)
    for causal in (False, True):
        fam.paged_attention_weights(b.q, torch.full(b.q.shape[:2], lse, device=cuda_device), b.k_cache, *b.where, w,
                                    causal, 64 ** -0.5, k_scale=b.k_scale)
        ops.check_device_status(cuda_device)
        assert not w.any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_rows_left_out_may_hold_anything(head_dim, fp8, bad, cuda_device):
    """A caller leaves rows out by lse = -inf: they give nothing to any key, whatever q holds there."""
    b = ref.Batch([130, 1, 40, 6], [500, 300, 40, 700], heads_q=8, heads_kv=2, head_dim=head_dim, page=32, fp8=fp8,
                  device=cuda_device, seed=8)
    for causal in (False, True):
        lse = ref_w.logsumexps(b, causal, head_dim ** -0.5)
        out = torch.rand(lse.shape, generator=torch.Generator().manual_seed(1)) < 0.2
        out[:33] = False   # a query tile without such rows,
        out[64:96] = True  # and one of nothing else
        lse[out.to(lse.device)] = float("-inf")
        b.q[out.to(lse.device)] = bad
        for longest in (None, 1):
            _check(b, causal, lse=lse, max_q_len=longest)
        b.q[out.to(lse.device)] = 1.0


def test_decoding_rows_left_out(cuda_device):
    """... and in a step of single tokens, a whole sequence's among them."""
    b = ref.Batch([1] * 40, [1 + 37 * i for i in range(40)], heads_q=8, heads_kv=2, head_dim=128, device=cuda_device, seed=9)
    lse = ref_w.logsumexps(b, True, 0.1)
    lse[7], lse[8, 3], lse[20, ::2] = (float("-inf"),) * 3
    b.q[torch.isneginf(lse)] = float("nan")
    _check(b, lse=lse, scale=0.1, max_q_len=1)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("l", [-88.0, -88.6, 80.0, 86.5])
def test_the_largest_and_smallest_weights_are_alike_in_every_row(l, fp8, cuda_device):
    """One row of 32 gives exp(-l), wherever it is: 88.6 is past 127.5 ln 2, 88.72 would be infinite.  (The others give
    exp(-200) = 0.)"""
    b = ref.Batch([32], [300], heads_q=1, heads_kv=1, head_dim=64, page=64, fp8=fp8, device=cuda_device, seed=8)
    b.q.zero_()
    args = (b.k_cache, *b.where)
    for r in range(32):
        w = torch.zeros(b.k_cache.shape[:3], device=cuda_device)
        lse = torch.full((32, 1), 200.0, device=cuda_device)
        lse[r] = l
        fam.paged_attention_weights(b.q, lse, *args, w, False, 0.125, k_scale=b.k_scale)
        flat = ref.gather(w, b.table, 0, 300).double()
        want = torch.exp(torch.tensor(-l, dtype=torch.float64, device=cuda_device))
        # (the tolerance of paged_weights_ref.py)
        assert ((flat - want).abs() <= 2.0 ** -21 * (1 + abs(l)) * want + 2.0 ** -126).all(), r
