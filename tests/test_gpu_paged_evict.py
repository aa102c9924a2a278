"""Eviction from the paged cache: every position, byte and length as on the host (B200)."""
from __future__ import annotations

import pytest
import torch

import flash_attention_forward as fam
import paged_evict_ref as ref_e
import paged_ref as ref
from flash_attn_npu_b200 import build, ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _weights(shape, seed, kind="mixed"):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2.5 * torch.randn(shape, generator=g) - 3)
    if kind == "mixed":  # ties, zeros of both signs, and numbers that no sum of probabilities is
        pick = torch.rand(shape, generator=g)
        w = torch.where(pick < 0.3, (w * 8).round() / 8, w)
        w = torch.where(pick > 0.9, -w, w)
        w = torch.where((pick > 0.4) & (pick < 0.45), torch.full_like(w, -0.0), w)
        for k, x in enumerate((float("inf"), float("-inf"), float("nan"), 1e-42, -1e-42)):
            w = torch.where((pick > 0.5 + 0.01 * k) & (pick < 0.505 + 0.01 * k), torch.full_like(w, x), w)
    elif kind == "equal":
        w = torch.full(shape, 0.25)
    return w


def _check(b, weights, keep, recent, to_pages=False):
    held = [b.k_cache, b.v_cache, weights] + ([b.k_scale, b.v_scale] if b.fp8 else [])
    to = None
    if to_pages:  # pages that no sequence has
        seqs, per = b.table.shape[0], max(1, -(-keep // b.page))
        free = [i for i in range(b.k_cache.shape[0]) if i not in set(b.table.flatten().tolist())]
        to = torch.tensor(free[:seqs * per], dtype=torch.int32).view(seqs, per).flip(0).contiguous()
        to = to.to(b.table.device)
    want_lens, want_kept, want = ref_e.evict(held, weights, b.table, b.lens, keep, recent, to)
    lens, kept = fam.paged_cache_evict(b.k_cache, b.v_cache, weights, b.table, b.lens, keep, recent, b.k_scale,
                                       b.v_scale, to_table=to, return_kept=True)
    ops.check_device_status(b.table.device)
    assert torch.equal(lens.cpu(), want_lens)
    assert torch.equal(kept.cpu(), want_kept)
    for x, y in zip(held, want):
        assert torch.equal(ref_e.bits(x.cpu()).view(y.shape), y)
    return lens, kept


def _batch(lens, device, spare=2, **more):
    return ref.Batch([0] * len(lens), lens, device=device, spare=spare, **more)


@pytest.mark.parametrize("to_pages", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128, 256])
def test_lengths(head_dim, fp8, to_pages, cuda_device):
    lens = [0, 1, 99, 100, 101, 128, 500, 1300]
    b = _batch(lens, cuda_device, heads_kv=3, heads_q=3, head_dim=head_dim, fp8=fp8, spare=100, seed=head_dim)
    w = _weights(b.k_cache.shape[:3], head_dim).to(cuda_device)
    _check(b, w, 100, 17, to_pages)


@pytest.mark.parametrize("keep,recent", [(0, 0), (1, 0), (1, 1), (64, 0), (64, 64), (65, 1), (700, 699), (899, 0),
                                         (900, 5), (5000, 3)])
@pytest.mark.parametrize("to_pages", [False, True])
def test_budgets(keep, recent, to_pages, cuda_device):
    lens = [900, 3, 64, 901, 66]
    b = _batch(lens, cuda_device, heads_kv=2, heads_q=2, head_dim=64, spare=5 * 320, seed=keep)
    _check(b, _weights(b.k_cache.shape[:3], keep + recent).to(cuda_device), keep, recent, to_pages)


@pytest.mark.parametrize("kind", ["equal", "mixed", "spread"])
@pytest.mark.parametrize("seqs", [1, 3, 40])
def test_long_sequences_and_ties(kind, seqs, cuda_device):
    """One sequence is shared by a cluster; equal weights go by position."""
    lens = [20011 // seqs + 13 * i for i in range(seqs)]
    b = _batch(lens, cuda_device, heads_kv=2, heads_q=2, head_dim=64, page=64, seed=seqs)
    w = _weights(b.k_cache.shape[:3], seqs, kind).to(cuda_device)
    _check(b, w, 3001 // seqs, 100 // seqs)


def test_positions_beyond_shared_memory(cuda_device):
    """Keys that do not fit a CTA's shared memory: a table of 2^19 positions, a sequence of 460,000."""
    b = _batch([460001], cuda_device, heads_kv=1, heads_q=1, head_dim=16, page=1024, seed=1)
    w = _weights(b.k_cache.shape[:3], 3).to(cuda_device)
    _check(b, w, 30011, 11)
    b = _batch([60001] * 40, cuda_device, heads_kv=4, heads_q=4, head_dim=16, page=1024, seed=1)
    w = _weights(b.k_cache.shape[:3], 3).to(cuda_device)
    _check(b, w, 50021, 0)


@pytest.mark.parametrize("page", [8, 128, 1024])
@pytest.mark.parametrize("layout", ["heads", "rows"])
def test_pages_and_layouts(page, layout, cuda_device):
    b = _batch([page, 3 * page + 1, 10 * page - 1], cuda_device, heads_kv=2, heads_q=2, head_dim=64, page=page,
               layout=layout, seed=page)
    w = _weights(b.k_cache.shape[:3], page)
    wide = torch.zeros(*w.shape[:2], w.shape[2] + 8)
    wide[..., :page] = w
    w = wide.to(cuda_device)[..., :page]  # rows of another pitch
    _check(b, w, 2 * page + 3, page // 2)


def test_what_stays_in_place_is_not_moved(cuda_device):
    """Falling weights: the first tokens stay, and only the recent ones move."""
    b = _batch([1000], cuda_device, heads_kv=1, heads_q=1, head_dim=64, page=1024, seed=2)
    w = torch.linspace(1, 0, 1024).view(1, 1, -1).expand(b.k_cache.shape[0], 1, -1).contiguous().to(cuda_device)
    _check(b, w, 600, 50)


def test_captured_step(cuda_device):
    """A replay goes by the lengths and weights of then; a second eviction finds what the first left."""
    b = _batch([400, 90, 700], cuda_device, heads_kv=2, heads_q=2, head_dim=64, seed=3)
    w = _weights(b.k_cache.shape[:3], 9, "spread").to(cuda_device)
    fam.paged_cache_evict(b.k_cache, b.v_cache, w, b.table, b.lens, 800, 10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens, kept = fam.paged_cache_evict(b.k_cache, b.v_cache, w, b.table, b.lens, 120, 10, return_kept=True)
    for turn in range(2):
        held = [b.k_cache, b.v_cache, w]
        want_lens, want_kept, want = ref_e.evict(held, w, b.table, b.lens, 120, 10)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lens.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
        for x, y in zip(held, want):
            assert torch.equal(ref_e.bits(x.cpu()).view(y.shape), y)
        b.lens -= 40
        w.copy_(_weights(w.shape, 10).to(cuda_device))


def test_pages_that_are_none_are_reported(cuda_device):
    b = _batch([400, 90], cuda_device, heads_kv=2, heads_q=2, head_dim=64, seed=3)
    w = _weights(b.k_cache.shape[:3], 9, "spread").to(cuda_device)
    table = b.table.clone()
    table[0, 3] = -7
    for where, to in ((table, None), (b.table, table[:, :8].contiguous()), (b.table, table[:, :2].contiguous())):
        fam.paged_cache_evict(b.k_cache.clone(), b.v_cache.clone(), w.clone(), where, b.lens, 100, 10, to_table=to)
        with pytest.raises(RuntimeError, match="page"):
            ops.check_device_status(cuda_device)
    ops.check_device_status(cuda_device)


@pytest.mark.parametrize("cols", [0, 1, 16])
@pytest.mark.parametrize("lens", [[5000], [70, 3000], [5000] * 40])
def test_a_table_too_narrow_for_what_stays_is_reported(lens, cols, cuda_device):
    """Also where it ends with a chunk of ranks (of K and V 128, of weights and scales 2048)."""
    b = _batch(lens, cuda_device, heads_kv=2, heads_q=2, head_dim=128, page=128, spare=16 * len(lens), seed=4)
    w = _weights(b.k_cache.shape[:3], 9, "spread").to(cuda_device)
    free = [i for i in range(b.k_cache.shape[0]) if i not in set(b.table.flatten().tolist())]
    to = torch.tensor(free[:cols * len(lens)], dtype=torch.int32, device=cuda_device).view(len(lens), cols)
    fam.paged_cache_evict(b.k_cache, b.v_cache, w, b.table, b.lens, 4096, 10, to_table=to)
    with pytest.raises(RuntimeError, match="page"):
        ops.check_device_status(cuda_device)
    # what fits is no matter: the same call with a budget of as many tokens as the table has places
    fam.paged_cache_evict(b.k_cache, b.v_cache, w, b.table, b.lens, cols * 128, 0, to_table=to)
    ops.check_device_status(cuda_device)


@pytest.mark.parametrize("kind", ["mixed", "equal"])
def test_positions_beyond_the_shared_memory_of_a_cluster(kind, cuda_device):
    """16 blocks hold 43,008 keys each: here they read 6,992 each from memory in every pass."""
    b = _batch([800001], cuda_device, heads_kv=1, heads_q=1, head_dim=16, page=1024, seed=1)
    w = _weights(b.k_cache.shape[:3], 3, kind).to(cuda_device)
    _check(b, w, 30011, 11)


@pytest.mark.parametrize("seqs", [1, 6, 48])
def test_tables_wider_than_their_sequences(seqs, cuda_device):
    """The plan goes by the table's width: clusters whose last blocks have nothing, for short sequences."""
    b = _batch([40 + 61 * i for i in range(seqs)], cuda_device, heads_kv=2, heads_q=2, head_dim=64, page=64, seed=seqs)
    wide = torch.full((seqs, 2048), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :b.table.shape[1]] = b.table
    before = [x.clone() for x in (b.k_cache, b.v_cache)]
    w = _weights(b.k_cache.shape[:3], 9).to(cuda_device)
    first = w.clone()
    narrow = b.table
    b.table = wide
    lens, kept = _check(b, w, 150, 20)
    # columns of the same table give the same
    b.k_cache, b.v_cache, b.table = *before, wide[:, :narrow.shape[1]]
    again = _check(b, first, 150, 20)
    assert torch.equal(again[0], lens) and torch.equal(again[1], kept)


@pytest.mark.parametrize("head_dim", [64, 128])
def test_captured_long_context(head_dim, cuda_device):
    """Clusters, tickets and flags: every replay finds them as the first did."""
    b = _batch([60000, 41000], cuda_device, heads_kv=2, heads_q=2, head_dim=head_dim, page=64, seed=3)
    w = _weights(b.k_cache.shape[:3], 9, "spread").to(cuda_device)
    fam.paged_cache_evict(b.k_cache.clone(), b.v_cache.clone(), w.clone(), b.table, b.lens, 9000, 10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens, kept = fam.paged_cache_evict(b.k_cache, b.v_cache, w, b.table, b.lens, 9000, 10, return_kept=True)
    for turn in range(3):
        held = [b.k_cache, b.v_cache, w]
        want_lens, want_kept, want = ref_e.evict(held, w, b.table, b.lens, 9000, 10)
        graph.replay()
        torch.cuda.synchronize()
        ops.check_device_status(cuda_device)
        assert torch.equal(lens.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
        for x, y in zip(held, want):
            assert torch.equal(ref_e.bits(x.cpu()).view(y.shape), y)
        b.lens -= 9000
