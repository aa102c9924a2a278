"""Paged attention over float8 caches whose scales lie far apart, or are no powers of two, and bf16 queries of
unequal channels.

The tolerance is that of tests/paged_ref.py without its allowance in units of the sequence's largest value, which
would hide what is looked for here: values that a few large rows make small.  With u = eps / 2,

    |out - ref| <= (u_p + r + 2 e) A + u |ref| + floor sum_j |v_j| ,   A = sum_j p_j |v_j| ,

sums over the keys that the row may attend to, and beside what is explained there
  * floor: a probability below fp16's normal numbers is off by at most half a step, 2^-25.  In the row kernel p carries
    2^10 and a ratio of scales of at least 2^-8, and some key of every warp has p = 1 before the division by l, so
    that is 2^-27; in the tile kernel with fp16 queries p carries 2^7: 2^-32; 0 with bf16 queries;
  * r: in the tile kernel code * scale is rounded to q's type, u, where the product does not fit it; the same of the
    keys adds u sum_d |q_d k_d| to the logit's error;
  * the fp32 sum over the keys: 16 or 32 keys a step, each step off by at most 2^-23 A;
  * fp16 has a step of 2^-24 below its normal numbers, where u |x| is less than half of it: an output there is off by
    up to 2^-25, and so is code * scale in the tile kernel with fp16 queries (these caches are quantised from fp32
    values, so it need not be one of fp16), which the p_j, summing to 1, carry over as it is.
"""
from __future__ import annotations

import pytest
import torch

import flash_attention_forward as fam
import paged_ref as ref
from flash_attn_npu_b200 import build, ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


def _want(b, causal, scale, rounded):
    """(out, lse, tolerance of out, tolerance of lse); `rounded`: code * scale need not fit q's type."""
    total, hq, d = b.q.shape
    hk = b.k_cache.shape[1]
    group = hq // hk
    few = max(b.offsets.diff().tolist()) * group <= 32
    u = torch.finfo(b.q.dtype).eps / 2
    u_p = torch.finfo(FP16 if few else b.q.dtype).eps / 2
    floor = 2.0 ** -27 if few else 2.0 ** -32 if b.q.dtype == FP16 else 0.0
    r = u if rounded and not few else 0.0
    least = 0.0 if b.q.dtype == BF16 else 2.0 ** -25 if few else 2.0 ** -24
    res = [torch.zeros(total, hq, d, dtype=torch.float64, device=b.q.device) for _ in range(2)]
    res += [torch.zeros(total, hq, dtype=torch.float64, device=b.q.device) for _ in range(2)]
    for i, n in enumerate(b.lens.tolist()):
        a, z = b.offsets[i:i + 2].tolist()
        x = b.q[a:z].double().view(z - a, hk, group, d)
        k, v = (ref.dequantise(ref.gather(c, b.table, i, n), ref.gather(s, b.table, i, n))
                for c, s in ((b.k_cache, b.k_scale), (b.v_cache, b.v_scale)))
        last = torch.arange(z - a, device=x.device)[:, None] + n - (z - a) if causal else n
        seen = (torch.arange(n, device=x.device)[None] <= last).expand(z - a, n)
        s = (torch.einsum("ihgd,jhd->hgij", x, k) * scale).masked_fill(~seen, float("-inf"))
        size = (torch.einsum("ihgd,jhd->hgij", x.abs(), k.abs()) * abs(scale)).masked_fill(~seen, 0.0)
        m = torch.logsumexp(s, -1)
        p = torch.exp(s - m[..., None])
        out, big = (torch.einsum("hgij,jhd->hgid", p, y) for y in (v, v.abs()))
        e = ((d + 8) * 2.0 ** -23 + r) * size.amax(-1) + 2.0 ** -20
        tol = (u_p + r + (n / 16 + 2) * 2.0 ** -23 + 2 * e)[..., None] * big + u * out.abs()
        tol = tol + least + floor * torch.einsum("ij,jhd->hid", seen.double(), v.abs())[:, None]
        for x, y in zip(res, (out, tol, m, e + 2.0 ** -22 * m.abs())):
            x[a:z] = y.permute(2, 0, 1, *range(3, y.ndim)).reshape(x[a:z].shape)
    return res[0], res[2], res[1], res[3]


def _check(b, causal=True, scale=None, rounded=False):
    scale = b.q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, causal, scale, **b.scales, return_lse=True,
                                   max_q_len=max(b.offsets.diff().tolist()))
    ops.check_device_status(b.q.device)
    want, want_lse, tol, tol_lse = _want(b, causal, scale, rounded)
    off = (out.double() - want).abs()
    assert (off <= tol).all(), ((off / tol)[~(off <= tol)]).max().item()
    assert ((lse.double() - want_lse).abs() <= tol_lse).all()


def _set(b, name, seq, at, rows):
    """Tokens `at` of sequence `seq` become `rows` [len(at), heads, D], as the cache's writer leaves them."""
    code, scale = ref.quantise(rows)
    at = torch.tensor(at)
    page, row = b.table.cpu()[seq, at // b.page].long(), at % b.page
    cache, held = (getattr(b, name + x) for x in ("_cache", "_scale"))
    cache.view(torch.uint8)[page, :, row] = code.view(torch.uint8).to(cache.device)
    held[page, :, row] = scale.to(held.device)


def _batch(counts, lens, gain, **kw):
    """Value rows of one size, about `gain`."""
    b = ref.Batch(counts, lens, fp8=True, heads_kv=2, heads_q=8, garbage=0.0, **kw)
    g = torch.Generator().manual_seed(1)
    for i, n in enumerate(lens):
        _set(b, "v", i, list(range(n)), gain * torch.randn(n, 2, b.q.shape[-1], generator=g))
    return b


COUNTS = [1, 2, 4, 8, 40]  # 4 to 160 rows a kv head: blocks of 8, 16 and 32 rows, tiles


@pytest.mark.parametrize("count", COUNTS)
@pytest.mark.parametrize("dtype,gain", [(BF16, 1e-3), (BF16, 1e-5), (BF16, 1e-7), (FP16, 2e-3)])
@pytest.mark.parametrize("zeros", ["first", "some"])
def test_rows_of_zeros_beside_small_ones(zeros, dtype, gain, count, cuda_device):
    """A row of zeros has scale 1, 2^10 to 2^30 times the others'."""
    lens = [600, max(count, 37)]
    b = _batch([count] * 2, lens, gain, head_dim=128, dtype=dtype, device=cuda_device)
    for i, n in enumerate(lens):
        at = [0] if zeros == "first" else list(range(3, n, 50))
        _set(b, "v", i, at, torch.zeros(len(at), 2, 128))
    _check(b)


@pytest.mark.parametrize("head_dim", [16, 32, 64, 256])
@pytest.mark.parametrize("count", [1, 8, 40])
def test_rows_of_zeros_at_every_head_dim(head_dim, count, cuda_device):
    b = _batch([count], [1000], 1e-6, head_dim=head_dim, dtype=BF16, device=cuda_device)
    _set(b, "v", 0, [0, 500], torch.zeros(2, 2, head_dim))
    _check(b)


@pytest.mark.parametrize("count", COUNTS[1:])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 40])
def test_large_values_that_the_mask_hides(size, count, cuda_device):
    """The last token's values are large: the rows before it do not see them."""
    b = _batch([count] * 2, [400, 129], 0.5, head_dim=64, dtype=BF16, device=cuda_device)
    for i, n in enumerate((400, 129)):
        _set(b, "v", i, [n - 1], size * torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(i)))
    _check(b)


@pytest.mark.parametrize("count", COUNTS)
@pytest.mark.parametrize("step", [1, 7, 20])
def test_scales_far_apart(step, count, cuda_device):
    """Value rows over 6 magnitudes, `step` powers of two from each to the next."""
    b = _batch([count] * 2, [700, 64], 1.0, head_dim=128, dtype=BF16, device=cuda_device)
    g = torch.Generator().manual_seed(2)
    for i, n in enumerate((700, 64)):
        x = torch.randn(n, 2, 128, generator=g) * torch.exp2(-step * torch.randint(0, 6, (n, 2, 1), generator=g))
        _set(b, "v", i, list(range(n)), x)
    _check(b)


@pytest.mark.parametrize("count", COUNTS)
def test_large_values_of_no_weight(count, cuda_device):
    """Rows 2^30 times the others, with logits far below theirs."""
    b = _batch([count], [700], 1.0, head_dim=64, dtype=BF16, device=cuda_device)
    g = torch.Generator().manual_seed(3)
    b.q = torch.rand(b.q.shape, generator=g).add(0.5).to(BF16).to(cuda_device)
    at = list(range(5, 700, 90))
    _set(b, "k", 0, at, torch.full((len(at), 2, 64), -10.0))
    _set(b, "v", 0, at, 2.0 ** 30 * torch.randn(len(at), 2, 64, generator=g))
    _check(b, scale=0.25)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("count", COUNTS)
def test_scales_that_are_no_powers_of_two(count, dtype, causal, cuda_device):
    for head_dim in (64, 256):
        b = ref.Batch([count] * 2, [500, 77], heads_q=8, heads_kv=2, head_dim=head_dim, dtype=dtype, fp8=True, garbage=0.0,
                      device=cuda_device, seed=head_dim)
        g = torch.Generator().manual_seed(4)
        for s in (b.k_scale, b.v_scale):
            s.mul_(torch.exp(0.5 * torch.randn(s.shape, generator=g)).to(cuda_device))
        _check(b, causal, rounded=True)

@pytest.mark.parametrize("count", COUNTS)
@pytest.mark.parametrize("low", [2.0 ** -10, 2.0 ** -18])
def test_queries_of_unequal_channels(low, count, cuda_device):
    """One channel of the queries is 2^20 or 2^28 times the others, and meets keys that are 0 there."""
    b = _batch([count], [300], 1.0, head_dim=64, dtype=BF16, device=cuda_device)
    g = torch.Generator().manual_seed(5)
    q = low * torch.randn(b.q.shape, generator=g)
    q[..., 7] = 2.0 ** 10
    b.q = q.to(BF16).to(cuda_device)
    k = torch.randn(300, 2, 64, generator=g) / low
    k[..., 7] = 0
    _set(b, "k", 0, list(range(300)), k)
    _check(b, scale=0.25)
    b.q[..., 7] = 0  # every channel small
    _check(b, scale=0.25)


@pytest.mark.parametrize("count", COUNTS)
def test_queries_of_zeros_and_a_small_scale(count, cuda_device):
    """The logits are 0 however small the scale is, and what the mask hides stays hidden."""
    b = _batch([count], [300], 1.0, head_dim=64, dtype=BF16, device=cuda_device)
    b.q.zero_()
    _check(b, scale=1e-30)


@pytest.mark.parametrize("count", COUNTS)
@pytest.mark.parametrize("power", [-126, -100, 60, 100])
def test_scales_at_the_ends_of_their_range(power, count, cuda_device):
    """Values at either end, and keys there too, with queries that bring the logits back."""
    b = ref.Batch([count] * 2, [500, 77], heads_q=8, heads_kv=2, head_dim=64, dtype=BF16, fp8=True, garbage=0.0,
                  device=cuda_device, seed=6)
    g = torch.Generator().manual_seed(7)
    b.v_scale = (2.0 ** power * (1 + torch.rand(b.v_scale.shape, generator=g))).to(cuda_device)
    _check(b, rounded=True)
    if power > -126:
        b.k_scale *= 2.0 ** power
        b.q *= 2.0 ** -power
        _check(b, rounded=True)


@pytest.mark.parametrize("count", COUNTS)
def test_scales_of_0_count_as_values_of_0(count, cuda_device):
    """Once each, also in tiles that are taken in several turns."""
    b = _batch([count], [500], 1e-5, head_dim=64, dtype=BF16, device=cuda_device)
    _set(b, "v", 0, list(range(5, 500, 16)), torch.zeros(31, 2, 64))
    at = torch.arange(0, 500, 7)
    page, row = b.table.cpu()[0, at // b.page].long(), at % b.page
    b.v_scale[page.to(cuda_device), :, row.to(cuda_device)] = 0
    _check(b)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("kind", ["subnormal", "any bits"])
@pytest.mark.parametrize("count", COUNTS)
def test_scales_outside_their_range_stay_within_their_sequence(count, kind, head_dim, cuda_device):
    """Whatever is found in place of scales, the call ends, and the other sequences are as they were."""
    b = ref.Batch([count] * 3, [300, 700, 129], heads_q=8, heads_kv=2, head_dim=head_dim, dtype=BF16, fp8=True, garbage=0.0,
                  device=cuda_device, seed=8)
    call = lambda: fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales, max_q_len=count)  # noqa: E731
    want = call()
    g = torch.Generator().manual_seed(9)
    pages = b.table[1][b.table[1] >= 0].long()
    for s in (b.k_scale, b.v_scale):
        bits = torch.randint(1, 1 << 23, (len(pages), *s.shape[1:]), generator=g, dtype=torch.int64)
        if kind == "any bits":
            bits = torch.randint(-2 ** 31, 2 ** 31, bits.shape, generator=g, dtype=torch.int64)
        s[pages] = bits.to(torch.int32).view(torch.float32).to(cuda_device)
    out = call()
    ops.check_device_status(cuda_device)
    assert torch.equal(out[:count], want[:count]) and torch.equal(out[2 * count:], want[2 * count:])
