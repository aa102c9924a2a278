"""The paged attention kernels where their division of work, copies and stores can go wrong: sequences cut among
CTAs at any length, tiles worked on by one or both sides, many sequences shorter than a copy, shared pages,
outputs of odd alignment, caches beyond 32-bit offsets.  Tolerances are those of tests/paged_ref.py."""
from __future__ import annotations

import os
import random
import subprocess
import sys

import pytest
import torch

import flash_attention_forward as fam
import paged_ref as ref
from conftest import REPO
from flash_attn_npu_b200 import build, ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _check(b, causal=True, max_q_len=None, **given):
    scale = b.q.shape[-1] ** -0.5
    out, lse = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, causal, scale, **b.scales,
                                   max_q_len=max_q_len, return_lse=True, **given)
    ops.check_device_status(b.q.device)
    want, want_lse, tol, tol_lse = ref.attention(b.q, b.k_cache, b.v_cache, *b.where, causal, scale, **b.scales,
                                                 max_q_len=max_q_len)
    n = int(b.offsets[-1])
    assert torch.equal(torch.isfinite(lse[:n]), torch.isfinite(want_lse[:n]))
    assert ((out.double() - want).abs()[:n] <= tol[:n]).all()
    live = torch.isfinite(want_lse[:n])
    assert ((lse.double() - want_lse).abs()[:n] <= tol_lse[:n])[live].all()
    return out, lse


def _widened(b, columns=4096):
    """The page table as a slice of a wide one: nothing is known of the lengths, so items may be cut."""
    wide = torch.full((b.table.shape[0], columns), -1, dtype=torch.int32, device=b.table.device)
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide
    return b


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("head_dim", [16, 64, 128, 256])
@pytest.mark.parametrize("rows", [1, 8, 60, 200])
def test_cut_anywhere(rows, head_dim, fp8, cuda_device):
    """Few sequences of drawn lengths behind a wide table: items of one to many parts, with empty steps at cuts."""
    rng = random.Random(100 * rows + head_dim + fp8)
    for turn in range(3):
        seqs = rng.choice([1, 2, 3, 5, 9])
        counts = [rng.randint(1, rows) for _ in range(seqs)]
        lens = [max(c, int(2 ** rng.uniform(0, 12.5))) for c in counts]
        b = ref.Batch(counts, lens, heads_q=rng.choice([2, 4, 10]), heads_kv=2, head_dim=head_dim,
                      page=rng.choice([8, 16, 64, 256]), fp8=fp8, dtype=rng.choice([BF16, FP16]), device=cuda_device,
                      seed=turn)
        _check(_widened(b), causal=turn != 1, max_q_len=max(counts))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("wide", [False, True])
def test_lone_tiles_of_every_length(wide, head_dim, fp8, cuda_device):
    """Blocks with tokens for one tile only, 1 to 24 key tiles, ending on, before and behind a tile's edge."""
    lens = [128 * n + d for n, d in zip(range(1, 25), [0, -1, 1, 64, -100, 5] * 4)]
    b = ref.Batch([11] * len(lens), lens, heads_q=4, heads_kv=1, head_dim=head_dim, page=32, fp8=fp8,
                  device=cuda_device, seed=head_dim)
    _check(_widened(b) if wide else b, max_q_len=11)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [8, 128, 1024])
@pytest.mark.parametrize("count", [1, 12])
def test_many_short_sequences(count, page, fp8, cuda_device):
    """Fewer keys than one copy holds, so that most producer warps have nothing to copy."""
    lens = [max(count, 1 + 7 * i % 23) for i in range(300)]
    for head_dim in (64, 128):
        b = ref.Batch([count] * 300, lens, heads_q=4, heads_kv=1, head_dim=head_dim, page=page, fp8=fp8, spare=1,
                      device=cuda_device, seed=page)
        _check(_widened(b, 64), max_q_len=count)


@pytest.mark.parametrize("heads", [(160, 1), (129, 1), (128, 1), (66, 2)])
def test_large_groups(heads, cuda_device):
    for fp8 in (False, True):
        b = ref.Batch([1, 3, 40], [300, 3, 77], heads_q=heads[0], heads_kv=heads[1], head_dim=64, fp8=fp8,
                      device=cuda_device, seed=heads[0])
        _check(b)
        _check(b, max_q_len=1)


@pytest.mark.parametrize("fp8", [False, True])
def test_shared_and_repeated_pages(fp8, cuda_device):
    """Two sequences with a common prefix, and one that names a page twice."""
    for counts in ([1, 1, 1], [70, 90, 40]):
        b = ref.Batch(counts, [500, 480, 300], heads_q=4, heads_kv=2, head_dim=128, page=32, fp8=fp8, garbage=0.0,
                      device=cuda_device, seed=3)
        b.table[1, :10] = b.table[0, :10]
        b.table[2, 1] = b.table[2, 0]
        _check(b)


@pytest.mark.parametrize("head_dim", [16, 64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_output_rows_aligned_to_16_bytes_only(head_dim, fp8, cuda_device):
    for counts in ([1, 3], [150, 40]):
        b = ref.Batch(counts, [700, 90], heads_q=4, heads_kv=2, head_dim=head_dim, fp8=fp8, device=cuda_device, pad=3)
        want, _ = _check(b)
        n = int(b.offsets[-1])
        flat = torch.full((b.total * 4 * (head_dim + 8) + 8,), 7.0, dtype=BF16, device=cuda_device)
        rows = flat[8:].view(b.total, 4, head_dim + 8)
        out, _ = _check(b, out=rows[..., :head_dim])
        assert torch.equal(out[:n], want[:n])
        assert (flat[:8] == 7).all() and (rows[..., head_dim:] == 7).all() and (rows[n:] == 7).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_cache_beyond_32_bit_offsets(fp8, cuda_device):
    """Pages at the end of a cache of more than 2^31 values: written, read back and attended to."""
    heads, page, head_dim = 8, 64, 128
    pages = (1 << 31) // (heads * page * head_dim) + 200
    dtype = ref.FP8 if fp8 else BF16
    cache = fam.paged_cache_empty(pages, page, heads, head_dim, dtype, cuda_device)
    small = ref.Batch([300, 1, 90], [300, 1, 90], heads_q=32, heads_kv=heads, head_dim=head_dim, page=page, fp8=fp8,
                      device=cuda_device, seed=8)
    shift = pages - small.k_cache.shape[0]
    table = torch.where(small.table >= 0, small.table + shift, small.table)
    scales = {"k_scale": cache[2], "v_scale": cache[3]}
    fam.paged_cache_write(*small.rows, *cache[:2], table, small.offsets, small.lens, **scales)
    fam.paged_cache_write(*small.rows, small.k_cache, small.v_cache, *small.where, **small.scales)
    for x, y in zip(fam.paged_cache_read(*cache[:2], table, small.offsets, small.lens, small.total, **scales),
                    fam.paged_cache_read(small.k_cache, small.v_cache, *small.where, small.total, **small.scales)):
        assert torch.equal(x, y)
    want, _ = _check(small)
    out = fam.paged_attention(small.q, *cache[:2], table, small.offsets, small.lens, True, head_dim ** -0.5, **scales)
    one = small.q[torch.tensor([299, 300, 390], device=cuda_device)]  # the last token of each, by the row kernel
    each = torch.arange(4, dtype=torch.int32, device=cuda_device)
    got = fam.paged_attention(one, *cache[:2], table, each, small.lens, True, head_dim ** -0.5, **scales)
    ops.check_device_status(cuda_device)
    assert torch.equal(out, want)
    plain, _, tol, _ = ref.attention(one, small.k_cache, small.v_cache, small.table, each, small.lens, True,
                                     head_dim ** -0.5, **small.scales)
    assert ((got.double() - plain).abs() <= tol).all()


_FIRST_CALL = """
import sys
sys.path[:0] = [{repo!r}, {repo!r} + "/tests"]
import torch
import flash_attention_forward as fam
import paged_ref as ref
from flash_attn_npu_b200 import ops
dev = torch.device("cuda", 0)
b = ref.Batch([{count}, 1], [3000, 200], heads_q=8, heads_kv=2, head_dim=128, fp8={fp8}, device=dev)
args = (b.q, b.k_cache, b.v_cache, *b.where, True, 0.1)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where, **b.scales)
    out, lse = fam.paged_attention(*args, **b.scales, return_lse=True)
    k, v = fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales)
graph.replay()
torch.cuda.synchronize()
want, _, tol, _ = ref.attention(*args, **b.scales)
assert ((out.double() - want).abs() <= tol).all()
again, _ = fam.paged_attention(*args, **b.scales, return_lse=True)
assert torch.equal(again, out)
ops.check_device_status(dev)
del graph
"""


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("count", [1, 100])
def test_first_calls_of_a_process_are_captured(count, fp8, cuda_device):
    """Nothing ran before the capture: no kernel was loaded, the device has no status word yet."""
    code = _FIRST_CALL.format(repo=str(REPO), count=count, fp8=fp8)
    res = subprocess.run([sys.executable, "-c", code], cwd=str(REPO), env=dict(os.environ), capture_output=True, text=True,
                         timeout=300)
    assert res.returncode == 0, res.stderr[-3000:]
