"""Plain 64-bit form of attention behind shared prefixes, and inputs for its tests.

The tolerance is that of `paged_ref.attention` over the joined keys.  Each probability is rounded to the
type of the products once, in the prefix's launch or the sequence's, and the parts are joined in fp32 with
weights that are off by the logsumexps' errors: 2 e more of A = sum_j p_j |v_j| for each of at most two
levels, and for each of the CTAs that share a level a few roundings of 2^-24, counted as 2^-18 in all.
"""
from __future__ import annotations

import torch

import paged_ref as ref


class PrefixBatch:
    """Sequences with `counts` new and `lens` own tokens; prefixes of `prefix_lens` tokens, shared by
    `members` packed rows each."""

    def __init__(self, counts, lens, prefix_lens, members, *, before=0, **more):
        n = len(counts)
        self.batch = ref.Batch(list(counts) + [0] * len(prefix_lens), list(lens) + list(prefix_lens), **more)
        b = self.batch
        self.q, self.k_cache, self.v_cache = b.q, b.k_cache, b.v_cache
        self.k_scale, self.v_scale, self.scales = b.k_scale, b.v_scale, b.scales
        self.table, self.offsets, self.lens = b.table[:n], b.offsets[:n + 1].clone(), b.lens[:n].clone()
        self.prefix_table, self.prefix_lens = b.table[n:], b.lens[n:].clone()
        self.prefix_offsets = (torch.tensor([0] + list(members)).cumsum(0) + before).to(torch.int32).to(b.q.device)
        self.total = b.total

    @property
    def prefix(self):
        return self.prefix_table, self.prefix_offsets, self.prefix_lens

    @property
    def where(self):
        return self.table, self.offsets, self.lens


def attention(x, causal, scale):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits; NaN where no sequence has a row."""
    q, dev = x.q, x.q.device
    total, hq, d = q.shape
    hk = x.k_cache.shape[1]
    group = hq // hk
    out = torch.full((total, hq, d), float("nan"), dtype=torch.float64, device=dev)
    lse = torch.full((total, hq), float("nan"), dtype=torch.float64, device=dev)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    u = torch.finfo(q.dtype).eps / 2
    offsets, lens = x.offsets.tolist(), x.lens.tolist()
    po, pl = x.prefix_offsets.tolist(), x.prefix_lens.tolist()

    def held(name, table, b, n):
        cache, s = getattr(x, name + "_cache"), getattr(x, name + "_scale")
        return ref.dequantise(ref.gather(cache, table, b, n), None if s is None else ref.gather(s, table, b, n))

    for b in range(len(lens)):
        count = offsets[b + 1] - offsets[b]
        ks, vs = held("k", x.table, b, lens[b]), held("v", x.table, b, lens[b])
        for t in range(offsets[b], offsets[b + 1]):
            n = lens[b] if not causal else max(0, min(lens[b], lens[b] - count + t - offsets[b] + 1))
            k, v = ks[:n], vs[:n]
            g = [g for g in range(len(pl)) if po[g] <= t < po[g + 1]]
            if g:
                k = torch.cat([held("k", x.prefix_table, g[0], pl[g[0]]), k])
                v = torch.cat([held("v", x.prefix_table, g[0], pl[g[0]]), v])
            if len(k) == 0:
                out[t], lse[t] = 0, float("-inf")
                continue
            y = q[t].double().view(hk, group, d)
            s = torch.einsum("hgd,jhd->hgj", y, k) * scale
            size = torch.einsum("hgd,jhd->hgj", y.abs(), k.abs()).amax(-1) * abs(scale)
            m = torch.logsumexp(s, -1)
            p = torch.exp(s - m[..., None])
            o = torch.einsum("hgj,jhd->hgd", p, v)
            e = (d + 8) * 2.0 ** -23 * size + 2.0 ** -20
            big = torch.einsum("hgj,jhd->hgd", p, v.abs())
            out[t] = o.reshape(hq, d)
            lse[t] = m.reshape(hq)
            tol[t] = ((u + 4 * e + 2.0 ** -18)[..., None] * big + u * o.abs()
                      + len(k) * 2.0 ** -32 * v.abs().amax()).reshape(hq, d)
            tol_lse[t] = (2 * e + 2.0 ** -22 * m.abs() + 2.0 ** -18).reshape(hq)
    return out, lse, tol, tol_lse
