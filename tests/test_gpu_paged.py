"""The paged cache's kernels against their 64-bit forms (tests/paged_ref.py has the tolerances)."""
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


def _same(a, b):
    """Bit-equal but for the bits of a NaN."""
    a, b = (x.float() if x.dtype == ref.FP8 else x for x in (a, b))
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(
        torch.nan_to_num(a, 0.0, 1e30, -1e30), torch.nan_to_num(b, 0.0, 1e30, -1e30))


def _check(b, causal=True, scale=None, max_q_len=None):
    scale = b.q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, causal, scale, **b.scales,
                                   max_q_len=max_q_len, return_lse=True)
    ops.check_device_status(b.q.device)
    want, want_lse, tol, tol_lse = ref.attention(b.q, b.k_cache, b.v_cache, *b.where, causal, scale, **b.scales,
                                                 max_q_len=max_q_len)
    n = int(b.offsets[-1])
    assert torch.equal(torch.isfinite(lse[:n]), torch.isfinite(want_lse[:n]))
    over = (out.double() - want).abs()[:n] - tol[:n]
    assert not (over > 0).any() and not torch.isnan(over).any(), over.max().item()
    live = torch.isfinite(want_lse[:n])
    over = ((lse.double() - want_lse).abs() - tol_lse)[:n][live]
    assert not (over > 0).any() and not torch.isnan(over).any(), over.max().item()
    assert torch.equal(lse[:n][~live], want_lse[:n][~live].float())
    return out, lse


# ------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128, 256])
def test_decode_ragged(head_dim, dtype, fp8, cuda_device):
    lens = [1, 7, 8, 9, 127, 128, 129, 255, 257, 600, 1, 1000]
    _check(ref.Batch([1] * len(lens), lens, heads_q=8, heads_kv=2, head_dim=head_dim, page=16, dtype=dtype,
                     fp8=fp8, device=cuda_device, seed=head_dim), max_q_len=1)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128, 256])
def test_chunks_ragged(head_dim, fp8, causal, cuda_device):
    counts = [5, 0, 1, 33, 64, 130, 300]
    lens = [5, 40, 1, 200, 64, 513, 900]
    _check(ref.Batch(counts, lens, heads_q=6, heads_kv=2, head_dim=head_dim, page=32, fp8=fp8,
                     dtype=FP16 if head_dim in (32, 128) else BF16, device=cuda_device, seed=1), causal)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("fp8", [False, True])
def test_page_sizes(page, fp8, cuda_device):
    _check(ref.Batch([1, 20, 3], [page, 2 * page + 5, 3 * page - 1] if page > 8 else [8, 21, 23],
                     head_dim=128, page=page, fp8=fp8, device=cuda_device, seed=2))


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (5, 5), (7, 1), (8, 1), (16, 1), (17, 1), (14, 2), (64, 2), (40, 1)])
@pytest.mark.parametrize("fp8", [False, True])
def test_head_groups(heads, fp8, cuda_device):
    _check(ref.Batch([1, 9, 2], [300, 77, 2], heads_q=heads[0], heads_kv=heads[1], head_dim=64, fp8=fp8,
                     device=cuda_device, seed=3))
    _check(ref.Batch([1, 150, 2], [300, 377, 2], heads_q=heads[0], heads_kv=heads[1], head_dim=128, fp8=fp8,
                     device=cuda_device, seed=3))


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_rows_without_keys(head_dim, fp8, cuda_device):
    """Empty sequences, chunks longer than what the cache holds, sequences without new tokens."""
    b = ref.Batch([1, 200, 0, 40, 3], [0, 0, 100, 10, 3], head_dim=head_dim, fp8=fp8, device=cuda_device, seed=4)
    out, lse = _check(b, True)
    assert (out[:201] == 0).all() and torch.isneginf(lse[:201]).all()
    assert torch.isneginf(lse[201:231]).all() and torch.isfinite(lse[231:]).all()
    _check(b, False)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_long_context_few_heads(head_dim, fp8, cuda_device):
    """One sequence is shared among many CTAs; also one whose tail is a single key."""
    _check(ref.Batch([1], [40001], heads_q=8, heads_kv=1, head_dim=head_dim, page=64, fp8=fp8, device=cuda_device,
                     seed=5), max_q_len=1)
    _check(ref.Batch([3, 1], [20000, 16385], heads_q=8, heads_kv=1, head_dim=head_dim, page=256, fp8=fp8,
                     device=cuda_device, seed=6), max_q_len=3)
    _check(ref.Batch([150], [6000], heads_q=8, heads_kv=1, head_dim=head_dim, page=64, fp8=fp8, device=cuda_device,
                     seed=7))


@pytest.mark.parametrize("fp8", [False, True])
def test_many_sequences(fp8, cuda_device):
    """More sequences than a CTA has threads, some without tokens."""
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(1, 60, (1500,), generator=g).tolist()
    counts = [min(n, int(c)) for n, c in zip(lens, torch.randint(0, 4, (1500,), generator=g))]
    _check(ref.Batch(counts, lens, head_dim=64, page=16, fp8=fp8, device=cuda_device, seed=8))


@pytest.mark.parametrize("causal", [False, True])
def test_chunk_from_nothing(causal, cuda_device):
    """Prompts: the cache holds nothing but the chunk."""
    for d, dtype in ((128, BF16), (64, FP16)):
        _check(ref.Batch([700, 257, 128, 1], [700, 257, 128, 1], heads_q=8, heads_kv=2, head_dim=d, dtype=dtype,
                         device=cuda_device, seed=9), causal)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
@pytest.mark.parametrize("fp8", [False, True])
def test_scales(scale, fp8, cuda_device):
    _check(ref.Batch([1, 40, 200], [300, 129, 400], head_dim=64, fp8=fp8, device=cuda_device, seed=10), True, scale)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("count", [1, 160])
def test_growing_maxima_and_unequal_values(count, fp8, cuda_device):
    """Each key's logit is above the last one's, and value rows spread over 2^30."""
    b = ref.Batch([count], [700], heads_q=4, heads_kv=1, head_dim=64, fp8=fp8, dtype=BF16, device=cuda_device, seed=11)
    for at in range(700):
        page, row = int(b.table[0, at // b.page]), at % b.page
        k = torch.full((64,), at / 100.0).to(BF16)
        v = (torch.randn(64, generator=torch.Generator().manual_seed(at)) * 2.0 ** (15 - at % 31)).to(BF16)
        if fp8:
            for x, c, s in ((k, b.k_cache, b.k_scale), (v, b.v_cache, b.v_scale)):
                code, sc = ref.quantise(x)
                c[page, 0, row], s[page, 0, row] = code.to(cuda_device), sc.to(cuda_device)
        else:
            b.k_cache[page, 0, row], b.v_cache[page, 0, row] = k.to(cuda_device), v.to(cuda_device)
    b.q = torch.rand(b.q.shape, generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda_device)
    _check(b, True, 0.05)


@pytest.mark.parametrize("fp8", [False, True])
def test_layouts(fp8, cuda_device):
    """A cache with the rows outside the heads, q cut from a larger tensor, wide tables, given outputs."""
    b = ref.Batch([1, 30, 140], [500, 77, 300], heads_q=4, heads_kv=2, head_dim=128, page=16, fp8=fp8, layout="rows",
                  device=cuda_device, seed=12, pad=5)
    wide = torch.full((3, 100), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide[:, :b.table.shape[1] + 3]
    mixed = torch.randn(b.total, 8, 128, device=cuda_device).to(BF16)
    mixed[:, :4] = b.q
    b.q = mixed[:, :4]
    want, want_lse = _check(b)
    out = torch.full((b.total, 6, 128), 7.0, dtype=BF16, device=cuda_device)
    lse = torch.full((b.total, 4), 7.0, device=cuda_device)
    n = int(b.offsets[-1])
    fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 128 ** -0.5, **b.scales, out=out[:, 1:5], lse=lse)
    assert torch.equal(out[:n, 1:5], want[:n]) and torch.equal(lse[:n], want_lse[:n])
    assert (out[n:] == 7).all() and (lse[n:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 5] == 7).all()
    odd = torch.randn(b.total, 4, 131, device=cuda_device).to(BF16)[..., 1:129]  # rows that are not aligned
    odd.copy_(b.q)
    again = fam.paged_attention(odd, b.k_cache, b.v_cache, *b.where, True, 128 ** -0.5, **b.scales)
    assert torch.equal(again[:n], want[:n])


def test_max_q_len_is_only_a_hint(cuda_device):
    b = ref.Batch([1, 300, 20], [50, 400, 600], heads_q=8, heads_kv=2, head_dim=128, device=cuda_device, seed=13)
    for hint in (None, 1, 2, 40, 300, 100000):
        _check(b, max_q_len=hint)


@pytest.mark.parametrize("fp8", [False, True])
def test_repeats_bit_for_bit(fp8, cuda_device):
    b = ref.Batch([1, 1, 200, 8], [9000, 33, 5000, 2000], heads_q=8, heads_kv=2, head_dim=128, page=64, fp8=fp8,
                  device=cuda_device, seed=14)
    first = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales, return_lse=True)
    for _ in range(20):
        again = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_nan_and_inf_inside_a_sequence_show(cuda_device):
    b = ref.Batch([1, 1], [300, 300], heads_q=2, heads_kv=1, head_dim=64, device=cuda_device, seed=15)
    b.v_cache[int(b.table[0, 3]), 0, 2, 5] = float("nan")
    out, lse = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, return_lse=True)
    assert torch.isnan(out[0, :, 5]).all() and torch.isfinite(out[0, :, :5]).all()
    assert torch.isfinite(out[1]).all() and torch.isfinite(lse).all()
    b.k_cache[int(b.table[0, 3]), 0, 2, 5] = float("nan")
    out, lse = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, return_lse=True)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_bad_tables_are_reported(head_dim, fp8, cuda_device):
    """Pages outside the cache and lengths outside the table are not followed; other sequences stand."""
    for count in (1, 200):
        b = ref.Batch([count, count, count], [400, 300, 500], head_dim=head_dim, fp8=fp8, device=cuda_device, seed=16)
        want, _ = _check(b)
        good_table, good_lens = b.table.clone(), b.lens.clone()
        for page in (-1, b.k_cache.shape[0], 2 ** 31 - 1, -2 ** 31):
            b.table[1, 2] = page
            out = fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, head_dim ** -0.5, **b.scales)
            with pytest.raises(RuntimeError, match="page"):
                ops.check_device_status(cuda_device)
            assert torch.equal(out[:count], want[:count]) and torch.equal(out[2 * count:], want[2 * count:])
        b.table = good_table
        for n in (-5, 10 ** 6, 2 ** 31 - 1):
            b.lens[1] = n
            fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, head_dim ** -0.5, **b.scales)
            with pytest.raises(RuntimeError, match="page"):
                ops.check_device_status(cuda_device)
        b.lens = good_lens
        b.offsets[-1] = b.total + 1000
        fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, head_dim ** -0.5, **b.scales)
        with pytest.raises(RuntimeError, match="page"):
            ops.check_device_status(cuda_device)
    ops.check_device_status(cuda_device)


# ------------------------------------------------------------------------------ write and read
def _plain_write(b, k, v, skip=None):
    got = [b.k_cache.clone(), b.v_cache.clone()]
    scales = [None, None] if not b.fp8 else [b.k_scale.clone(), b.v_scale.clone()]
    for x, c, s in ((k, got[0], scales[0]), (v, got[1], scales[1])):
        codes, sc = ref.quantise(x) if b.fp8 else (x, None)
        raw, flat = (codes.view(torch.uint8), c.view(torch.uint8)) if b.fp8 else (codes, c)
        for i in range(len(b.lens)):
            if i == skip:
                continue
            pos = torch.tensor(list(ref.positions(b.offsets, b.lens, i)), dtype=torch.long, device=x.device)
            page, row = b.table[i, pos // b.page].long(), pos % b.page
            at = slice(int(b.offsets[i]), int(b.offsets[i + 1]))
            flat[page, :, row] = raw[at]
            if s is not None:
                s[page, :, row] = sc[at]
    return got + scales


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("head_dim,heads,page", [(16, 1, 8), (32, 3, 16), (64, 2, 64), (128, 8, 16), (256, 5, 1024)])
def test_write_and_read_back(head_dim, heads, page, dtype, fp8, cuda_device):
    b = ref.Batch([1, 0, 33, 17, 200], [1, 9, 100, 17, 1300], heads_q=heads, heads_kv=heads, head_dim=head_dim,
                  page=page, dtype=dtype, fp8=fp8, device=cuda_device, seed=20, pad=3)
    k, v = b.rows
    k[3] = 0                       # a row of zeros
    k[4, 0, 1] = float("inf")
    k[5, 0, 3], k[5, 0, 4] = float("nan"), float("-inf")
    k[6] *= 2.0 ** -20             # subnormal in fp16
    v[0] = 448.0                   # at the borders of a scale
    v[1, :, 0] = 7 * 2.0 ** 8
    v[2] = torch.nextafter(torch.tensor(448.0), torch.tensor(1000.0)).to(dtype)
    if dtype == BF16:
        k[7] = 2.0 ** -133         # subnormal even in fp32
        v[3] = torch.finfo(BF16).max
    want = _plain_write(b, k, v)
    # rows cut from a projection of q, k and v
    mixed = torch.randn(b.total, 2 * heads + 1, head_dim, device=cuda_device).to(dtype)
    mixed[:, 1:1 + heads], mixed[:, 1 + heads:] = k, v
    fam.paged_cache_write(mixed[:, 1:1 + heads], mixed[:, 1 + heads:], b.k_cache, b.v_cache, *b.where, **b.scales)
    ops.check_device_status(cuda_device)
    for got, w in zip([b.k_cache, b.v_cache, b.k_scale, b.v_scale], want):
        assert w is None or _same(got, w)
    # ... and back
    out = [torch.full((b.total, heads, head_dim), 7.0, dtype=dtype, device=cuda_device) for _ in range(2)]
    fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales, out=out)
    ops.check_device_status(cuda_device)
    n = int(b.offsets[-1])
    for x, got, name in ((k, out[0], "k"), (v, out[1], "v")):
        if fp8:
            code, scale = ref.quantise(x[:n])
            w = (code.float().double() * scale.double()[..., None]).to(dtype)
        else:
            w = x[:n]
        assert _same(got[:n], w), name
        assert (got[n:] == 7).all()
    if fp8:
        other = FP16 if dtype == BF16 else BF16
        got = fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales, dtype=other)
        code, scale = ref.quantise(v[:n])
        assert _same(got[1][:n], (code.float().double() * scale.double()[..., None]).to(other))


def test_write_many_sequences_and_layouts(cuda_device):
    g = torch.Generator().manual_seed(21)
    lens = torch.randint(1, 40, (1300,), generator=g).tolist()
    counts = [min(n, int(c)) for n, c in zip(lens, torch.randint(0, 3, (1300,), generator=g))]
    for layout in ("heads", "rows"):
        b = ref.Batch(counts, lens, head_dim=64, fp8=True, device=cuda_device, seed=21, layout=layout)
        want = _plain_write(b, *b.rows)
        odd = torch.randn(b.total, 2, 67, device=cuda_device).to(BF16)[..., 1:65]  # rows that are not aligned
        odd.copy_(b.rows[0])
        fam.paged_cache_write(odd, b.rows[1], b.k_cache, b.v_cache, *b.where, **b.scales)
        for got, w in zip([b.k_cache, b.v_cache, b.k_scale, b.v_scale], want):
            assert _same(got, w)


@pytest.mark.parametrize("fp8", [False, True])
def test_copy_reports_bad_tables(fp8, cuda_device):
    b = ref.Batch([4, 4, 4], [40, 40, 40], fp8=fp8, device=cuda_device, seed=22)
    b.table[1, 2] = b.k_cache.shape[0]
    want = _plain_write(b, *b.rows, skip=1)
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where, **b.scales)
    with pytest.raises(RuntimeError, match="page"):
        ops.check_device_status(cuda_device)
    assert _same(b.k_cache, want[0]) and _same(b.v_cache, want[1])
    got = fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, b.total, **b.scales)
    with pytest.raises(RuntimeError, match="page"):
        ops.check_device_status(cuda_device)
    assert (got[0][4:8] == 0).all() and (got[0][:4] != 0).any() and (got[0][8:] != 0).any()
    b.table[1, 2] = 0
    b.lens[1] = 3  # shorter than its chunk
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where, **b.scales)
    with pytest.raises(RuntimeError, match="page"):
        ops.check_device_status(cuda_device)


# ------------------------------------------------------------------------------ as it is used
@pytest.mark.parametrize("fp8", [False, True])
def test_prompt_then_decoding(fp8, cuda_device):
    """Prompts in chunks, then tokens one by one: every step agrees with the 64-bit form over the
    cache that the writes left, and the cache reads back as the tokens that went in."""
    g = torch.Generator().manual_seed(30)
    hq, hk, d, page = 8, 2, 128, 16
    prompts = [70, 5, 260]
    steps = [[40, 5, 100], [30, 0, 160], [1, 1, 1], [1, 1, 1], [1, 0, 1]]
    final = [sum(s[b] for s in steps) for b in range(3)]
    pages = sum(-(-n // page) for n in final)
    cache = fam.paged_cache_empty(pages + 1, page, hk, d, ref.FP8 if fp8 else BF16, cuda_device)
    table = torch.full((3, max(-(-n // page) for n in final)), -1, dtype=torch.int32)
    order = torch.randperm(pages + 1, generator=g)
    at = 0
    for b, n in enumerate(final):
        table[b, :-(-n // page)] = order[at:at - (-n // page)]
        at -= -n // page
    table = table.to(cuda_device)
    scales = {"k_scale": cache[2], "v_scale": cache[3]}
    lens, tokens = [0, 0, 0], [[], [], []]
    assert prompts == [sum(s[b] for s in steps[:2]) for b in range(3)]
    for counts in steps:
        lens = [n + c for n, c in zip(lens, counts)]
        offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(cuda_device)
        kv_lens = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
        mixed = torch.randn(sum(counts), hq + 2 * hk, d, generator=g).to(BF16).to(cuda_device)
        q, k, v = mixed[:, :hq], mixed[:, hq:hq + hk], mixed[:, hq + hk:]
        for b in range(3):
            tokens[b].append(k[int(offsets[b]):int(offsets[b + 1])])
        fam.paged_cache_write(k, v, cache[0], cache[1], table, offsets, kv_lens, **scales)
        out, lse = fam.paged_attention(q, cache[0], cache[1], table, offsets, kv_lens, True, d ** -0.5,
                                       max_q_len=max(counts), return_lse=True, **scales)
        want, want_lse, tol, tol_lse = ref.attention(q, cache[0], cache[1], table, offsets, kv_lens, True, d ** -0.5,
                                                     **scales)
        assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= tol_lse).all()
    offsets = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(cuda_device)
    got, _ = fam.paged_cache_read(cache[0], cache[1], table, offsets, kv_lens, sum(lens), **scales)
    all_k = torch.cat([x for t in tokens for x in t])
    if fp8:
        code, scale = ref.quantise(all_k)
        all_k = (code.float() * scale[..., None]).to(BF16)
    assert torch.equal(got, all_k)
    ops.check_device_status(cuda_device)


def test_agrees_with_dense_attention(cuda_device):
    """A prompt in a 16-bit cache, against the framework's own dense attention of the same tokens."""
    n, h, d = 500, 4, 128
    b = ref.Batch([n], [n], heads_q=h, heads_kv=h, head_dim=d, device=cuda_device, seed=31)
    k, v = fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, n)
    dense, dense_lse = fam.attention(*(x.transpose(0, 1)[None].contiguous() for x in (b.q, k, v)), True, d ** -0.5,
                                     return_lse=True)
    out, lse = _check(b)
    _, _, tol, tol_lse = ref.attention(b.q, b.k_cache, b.v_cache, *b.where, True, d ** -0.5)
    assert ((dense[0].transpose(0, 1) - out).double().abs() <= 2 * tol).all()
    assert ((dense_lse[0].T - lse).double().abs() <= 2 * tol_lse).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_two_graphs_and_another_stream(fp8, cuda_device):
    """Two captured steps and eager calls share no workspace; replays see new inputs and lengths."""
    mk = lambda seed, counts, lens: ref.Batch(counts, lens, heads_q=8, heads_kv=1, head_dim=128, page=64, fp8=fp8,  # noqa: E731
                                              device=cuda_device, seed=seed)
    a, z = mk(40, [1, 1], [6000, 3000]), mk(41, [150, 1], [4000, 9000])

    def step(b):
        fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where, **b.scales)
        return fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.09, **b.scales, return_lse=True)

    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        for b in (a, z):
            step(b)
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    graphs, outs = [], []
    for b in (a, z):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(b))
        graphs.append(graph)
    a.lens.copy_(torch.tensor([5500, 2999]))
    for b in (a, z):
        b.q.copy_(torch.randn(b.q.shape, device=cuda_device))
        for x in b.rows:
            x.copy_(torch.randn(x.shape, device=cuda_device))
    torch.cuda.synchronize(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    torch.cuda.synchronize(cuda_device)
    kept = [[x.clone() for x in o] for o in outs]
    for b, o in zip((a, z), kept):
        with torch.cuda.stream(side):
            e = step(b)
        torch.cuda.synchronize(cuda_device)
        assert torch.equal(o[0], e[0]) and torch.equal(o[1], e[1])
        want, _, tol, _ = ref.attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.09, **b.scales)
        assert ((o[0].double() - want).abs() <= tol).all()
    ops.check_device_status(cuda_device)
    del graphs


def test_empty_calls(cuda_device):
    b = ref.Batch([1], [10], device=cuda_device)
    none = torch.empty(0, dtype=torch.int32, device=cuda_device)
    out, lse = fam.paged_attention(b.q[:0], b.k_cache, b.v_cache, b.table[:0], b.offsets[:1], none, True, 0.1,
                                   return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    fam.paged_cache_write(b.rows[0][:0], b.rows[1][:0], b.k_cache, b.v_cache, *b.where)
    k, _ = fam.paged_cache_read(b.k_cache, b.v_cache, *b.where, 0)
    assert k.shape == (0, 2, 64)
    b.offsets.zero_()  # no sequence has a token: all rows are padding
    out = torch.full_like(b.q, 7.0)
    fam.paged_attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, out=out)
    fam.paged_cache_write(*b.rows, b.k_cache, b.v_cache, *b.where)
    ops.check_device_status(cuda_device)
    assert (out == 7).all()
