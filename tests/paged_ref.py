"""Plain 64-bit forms of the paged cache operators, and inputs for their tests.

Tolerances count roundings.  u = eps / 2 of the output's type is the largest relative error of one
rounding to it.  The kernels round each probability to 16 bits and the output once.  A probability is
rounded to the type of the products (u_p): that is q's, but fp16 where at most 32 query rows a kv
head meet a float8 cache, whose codes that kernel takes as fp16.  So

    |out - ref| <= (u_p + e) A + u |ref| + tiny,    A = sum_j p_j |v_j|
where e bounds the relative error of a probability from fp32 arithmetic: a logit is a sum of D
products accumulated in fp32, off by at most (D + 8) 2^-23 sum_d |q_d k_d| (truncating adders
counted as a whole step), the exponential and the scalings by a few 2^-22; the same bound, taken
twice, covers the sum l as well.  fp16 probabilities carry a factor of at least 2^7, so what falls
below fp16's subnormal step of 2^-24 loses at most 2^-32 of the row's largest: tiny = keys 2^-32
max |v|.
Without the factor u_p the same e bounds the logsumexp's absolute error, next to its own rounding.
"""
from __future__ import annotations

import torch

FP8 = torch.float8_e4m3fn


def quantise(x):
    """(codes, scales) of rows x[..., D]: the definition, step by step."""
    f = x.double()
    finite = torch.where(torch.isfinite(f), f.abs(), torch.zeros_like(f))
    top = finite.amax(-1)
    scale = torch.full_like(top, 2.0 ** -126)
    for e in range(-125, 129):  # the smallest power of two that is enough
        scale = torch.where(448 * scale < top, torch.full_like(top, 2.0 ** e), scale)
    scale = torch.where(top == 0, torch.ones_like(top), scale)
    y = torch.where(torch.isfinite(f), f / scale[..., None], torch.full_like(f, float("nan")))
    return y.float().to(FP8), scale.float()


def dequantise(cache, scale):
    x = cache.double() if cache.dtype != FP8 else cache.float().double()
    return x if scale is None else x * scale.double()[..., None]


def positions(offsets, lens, b):
    n = int(offsets[b + 1]) - int(offsets[b])
    return range(int(lens[b]) - n, int(lens[b]))


def gather(x, table, b, n):
    """Tokens 0 .. n - 1 of sequence b from x [pages, heads, page, ...]: [n, heads, ...]."""
    size = x.shape[2]
    pages = table[b, :-(-n // size)].long()
    return x[pages].transpose(1, 2).flatten(0, 1)[:n]


def attention(q, k_cache, v_cache, table, offsets, lens, causal, scale, k_scale=None, v_scale=None, max_q_len=None):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits; NaN where no sequence has a row."""
    dev = q.device
    total, hq, d = q.shape
    hk = k_cache.shape[1]
    group = hq // hk
    out = torch.full((total, hq, d), float("nan"), dtype=torch.float64, device=dev)
    lse = torch.full((total, hq), float("nan"), dtype=torch.float64, device=dev)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    u = torch.finfo(q.dtype).eps / 2
    few = min(max_q_len or total, total) * group <= 32 or scale <= 0 or group > 128
    half = q.dtype == torch.float16 or (k_cache.dtype == FP8 and few)
    u_p = torch.finfo(torch.float16 if half else torch.bfloat16).eps / 2
    offsets, lens = offsets.tolist(), lens.tolist()
    for b in range(len(lens)):
        a, z, n = offsets[b], offsets[b + 1], lens[b]
        count = z - a
        if count == 0:
            continue
        x = q[a:z].double().view(count, hk, group, d)
        k = dequantise(gather(k_cache, table, b, n), None if k_scale is None else gather(k_scale, table, b, n))
        v = dequantise(gather(v_cache, table, b, n), None if v_scale is None else gather(v_scale, table, b, n))
        s = torch.einsum("ihgd,jhd->hgij", x, k) * scale
        size = torch.einsum("ihgd,jhd->hgij", x.abs(), k.abs()) * abs(scale)
        if causal:
            i = torch.arange(count, device=dev)[:, None] + n - count
            s = s.masked_fill(torch.arange(n, device=dev)[None] > i, float("-inf"))
        if n == 0:
            o = torch.zeros((hk, group, count, d), dtype=torch.float64, device=dev)
            m = torch.full((hk, group, count), float("-inf"), dtype=torch.float64, device=dev)
            t, tl = torch.zeros_like(o), torch.zeros_like(m)
        else:
            m = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m)[..., None])
            o = torch.einsum("hgij,jhd->hgid", p, v)
            e = (d + 8) * 2.0 ** -23 * size.amax(-1) + 2.0 ** -20
            big = torch.einsum("hgij,jhd->hgid", p, v.abs())
            t = (u_p + 2 * e)[..., None] * big + u * o.abs() + n * 2.0 ** -32 * v.abs().amax()
            tl = e + 2.0 ** -22 * torch.where(torch.isfinite(m), m.abs(), torch.zeros_like(m))
        out[a:z] = o.permute(2, 0, 1, 3).reshape(count, hq, d)
        lse[a:z] = m.permute(2, 0, 1).reshape(count, hq)
        tol[a:z] = t.permute(2, 0, 1, 3).reshape(count, hq, d)
        tol_lse[a:z] = tl.permute(2, 0, 1).reshape(count, hq)
    return out, lse, tol, tol_lse


class Batch:
    """Sequences with `counts` new tokens and `lens` tokens each, over shuffled pages."""

    def __init__(self, counts, lens, *, heads_q=4, heads_kv=2, head_dim=64, page=16, dtype=torch.bfloat16,
                 fp8=False, device="cpu", seed=0, spare=2, layout="heads", garbage=float("nan"), pad=0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.dtype, self.fp8 = page, dtype, fp8
        per = [-(-n // page) for n in lens]
        pages = max(1, sum(per)) + spare
        order = torch.randperm(pages, generator=g)
        table = torch.full((len(lens), max([1] + per)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        shape = (pages, heads_kv, page, head_dim)
        held = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(per[b]):
                held[table[b, j], :min(page, n - j * page)] = True

        def cache(spread):
            x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[:3] + (1,), generator=g))
            x = x.to(dtype)
            # whatever lies outside the sequences must not matter
            hole = ~held[:, None, :, None]
            if not fp8:
                return x.masked_fill(hole, garbage), None
            code, scale = quantise(x)
            code = code.float().masked_fill(hole, garbage).to(FP8)
            return code, scale.masked_fill(hole[..., 0], garbage)

        self.k_cache, self.k_scale = cache(0.1)
        self.v_cache, self.v_scale = cache(0.5)
        self.table, self.held = table, held
        self.offsets = torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.total = int(self.offsets[-1]) + pad
        self.q = torch.randn(self.total, heads_q, head_dim, generator=g).to(dtype)
        self.rows = [torch.randn(self.total, heads_kv, head_dim, generator=g).to(dtype) for _ in range(2)]
        for name, x in list(vars(self).items()):
            if isinstance(x, torch.Tensor):
                setattr(self, name, x.to(device))
        self.rows = [x.to(device) for x in self.rows]
        if layout == "rows":  # [pages, page, heads, D] in memory
            self.k_cache, self.v_cache = (x.transpose(1, 2).contiguous().transpose(1, 2)
                                          for x in (self.k_cache, self.v_cache))

    @property
    def where(self):
        return self.table, self.offsets, self.lens

    @property
    def scales(self):
        return {"k_scale": self.k_scale, "v_scale": self.v_scale}
