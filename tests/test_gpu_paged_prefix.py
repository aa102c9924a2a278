"""Attention behind shared prefixes against its 64-bit form (B200)."""
from __future__ import annotations

import pytest
import torch

import flash_attention_forward as fam
import paged_prefix_ref as pre
import paged_ref as ref
from flash_attn_npu_b200 import build, ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _call(x, causal, scale, **more):
    return fam.paged_prefix_attention(x.q, x.k_cache, x.v_cache, *x.prefix, *x.where, causal, scale,
                                      return_lse=True, **x.scales, **more)


def _check(x, causal=True, scale=None, **more):
    scale = x.q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = _call(x, causal, scale, **more)
    ops.check_device_status(x.q.device)
    want, want_lse, tol, tol_lse = pre.attention(x, causal, scale)
    rows = slice(int(x.offsets[0]), int(x.offsets[-1]))
    live = torch.isfinite(want_lse[rows])
    assert torch.equal(torch.isfinite(lse[rows]), live)
    over = ((out.double() - want).abs() - tol)[rows]
    assert not (over > 0).any() and not torch.isnan(over).any(), over.max().item()
    over = ((lse.double() - want_lse).abs() - tol_lse)[rows][live]
    assert not (over > 0).any() and not torch.isnan(over).any(), over.max().item()
    assert torch.equal(lse[rows][~live], want_lse[rows][~live].float())
    assert (out[rows][~live] == 0).all()
    return out, lse


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128, 256])
def test_decoding(head_dim, dtype, fp8, cuda_device):
    lens = [1, 7, 130, 33, 257, 2, 64, 600, 1, 128, 9, 300]
    _check(pre.PrefixBatch([1] * 12, lens, [701], [12], heads_q=8, heads_kv=2, head_dim=head_dim, dtype=dtype,
                           fp8=fp8, device=cuda_device, seed=head_dim), max_q_len=1)


@pytest.mark.parametrize("rows", [1, 2, 7, 9, 33, 100])
@pytest.mark.parametrize("group", [1, 4])
def test_row_and_tile_kernels(rows, group, cuda_device):
    """Few and many rows that share a prefix; single tokens and chunks."""
    for count in (1, 3, 40):
        x = pre.PrefixBatch([count] * rows, [count + 5 * i for i in range(rows)], [1000], [count * rows],
                            heads_q=2 * group, heads_kv=2, head_dim=64, device=cuda_device, seed=rows)
        _check(x, max_q_len=count)
        _check(x)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_groups(causal, fp8, cuda_device):
    """Several prefixes: of one token, none, ends inside a page and a tile; sequences without rows, cut by
    a group's border, of no group, longer than what they hold."""
    x = pre.PrefixBatch([3, 0, 5, 1, 70, 4, 2], [10, 4, 5, 1, 60, 0, 200], [1, 257, 0, 640], [3, 4, 20, 40],
                        before=2, heads_q=6, heads_kv=2, head_dim=128, page=32, fp8=fp8, device=cuda_device,
                        seed=5, pad=9)
    _check(x, causal)
    _check(x, causal, max_q_len=70, max_prefix_q_len=40)
    _check(x, causal, max_q_len=1, max_prefix_q_len=1)


def test_rows_without_any_key(cuda_device):
    x = pre.PrefixBatch([4, 2], [2, 0], [0, 5], [5, 1], head_dim=64, device=cuda_device, seed=1)
    out, lse = _check(x)
    assert torch.isneginf(lse[:2]).all() and torch.isneginf(lse[4]).all() and torch.isfinite(lse[5]).all()


def test_no_prefixes_is_attention(cuda_device):
    x = pre.PrefixBatch([1, 9], [300, 77], [], [], head_dim=128, device=cuda_device, seed=2)
    _check(x)


def test_joined_sequence_agrees_with_one(cuda_device):
    """A prefix and what follows it, in pages of one sequence each, against `paged_attention` over both."""
    counts, own, pl, page = [1, 6, 1], [17, 40, 300], 512, 32
    x = pre.PrefixBatch(counts, own, [pl], [8], heads_q=8, heads_kv=2, head_dim=128, page=page,
                        device=cuda_device, seed=3)
    out, lse = _call(x, True, 0.1)
    table = torch.cat([x.prefix_table[:, :pl // page].expand(3, -1), x.table], 1).contiguous()
    want, want_lse = fam.paged_attention(x.q, x.k_cache, x.v_cache, table, x.offsets, x.lens + pl, True, 0.1,
                                         return_lse=True)
    torch.testing.assert_close(lse, want_lse, atol=1e-4, rtol=1e-5)
    assert (out.float() - want.float()).abs().max() < 2.0 ** -6 * x.v_cache[torch.isfinite(x.v_cache)].abs().max()


@pytest.mark.parametrize("heads", [(3, 1), (8, 8), (40, 1), (129, 1)])
def test_head_groups(heads, cuda_device):
    _check(pre.PrefixBatch([1, 9, 2], [30, 77, 2], [333], [12], heads_q=heads[0], heads_kv=heads[1], head_dim=64,
                           device=cuda_device, seed=3))


@pytest.mark.parametrize("scale", [-0.2, 0.0, 5.0])
def test_scales(scale, cuda_device):
    _check(pre.PrefixBatch([1, 1, 30], [30, 77, 40], [333], [32], head_dim=64, device=cuda_device, seed=3),
           scale=scale)


def test_long_prefix_is_shared_among_ctas(cuda_device):
    """One kv head: both levels are cut into many parts."""
    _check(pre.PrefixBatch([1], [4000], [50001], [1], heads_q=8, heads_kv=1, head_dim=128, page=64,
                           device=cuda_device, seed=6), max_q_len=1)
    _check(pre.PrefixBatch([2] * 20, [200 * i + 2 for i in range(20)], [30011], [40], heads_q=8, heads_kv=1,
                           head_dim=64, page=64, fp8=True, device=cuda_device, seed=6), max_q_len=2)


def test_outputs_given_and_rows_outside(cuda_device):
    x = pre.PrefixBatch([2, 3], [20, 30], [100], [9], head_dim=64, device=cuda_device, seed=4, pad=4)
    x.offsets += 2  # rows 0, 1 and 7, 8 belong to no sequence
    out, lse = torch.full_like(x.q, 7.0), torch.full(x.q.shape[:2], 7.0, device=cuda_device)
    got = _call(x, True, 0.125, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    assert (out[:2] == 7).all() and (out[7:] == 7).all() and (lse[:2] == 7).all() and (lse[7:] == 7).all()
    want, want_lse, tol, tol_lse = pre.attention(x, True, 0.125)
    assert ((out[2:7].double() - want[2:7]).abs() <= tol[2:7]).all()
    assert ((lse[2:7].double() - want_lse[2:7]).abs() <= tol_lse[2:7]).all()


def test_same_bits_every_time_and_in_a_graph(cuda_device):
    x = pre.PrefixBatch([1] * 40, [50 * i + 1 for i in range(40)], [5000, 3001], [25, 15], heads_q=16, heads_kv=4,
                        head_dim=128, device=cuda_device, seed=7)
    first = _call(x, True, 0.1, max_q_len=1)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(_call(x, True, 0.1, max_q_len=1), first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _call(x, True, 0.1, max_q_len=1)
    # lengths and queries are those of the replay
    x.lens -= 1
    x.lens.clamp_(min=1)
    x.prefix_lens -= 17
    x.q.mul_(0.5)
    graph.replay()
    want = _call(x, True, 0.1, max_q_len=1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_pages_that_are_none_are_reported(cuda_device):
    x = pre.PrefixBatch([1, 1], [20, 30], [100], [2], head_dim=64, device=cuda_device, seed=4)
    x.prefix_table = x.prefix_table.clone()
    x.prefix_table[0, 2] = 10 ** 6
    _call(x, True, 0.125)
    with pytest.raises(RuntimeError):
        ops.check_device_status(cuda_device)
    ops.check_device_status(cuda_device)
