"""Plain 64-bit form of the attention weights of cached tokens, with the tolerance of each.

A weight is a sum over rows i of p_ij = exp(s_ij - l_i).  The kernel's logit is a sum of D products
accumulated in fp32, off by at most (D + 8) 2^-23 sum_d |q_d k_d| (truncating adders counted as a whole
step); the scale, the key's scale, the logsumexp and their difference are rounded a few times each, 2^-21
(1 + |s| + |l|) in all, in which the exponential's own error is.  That is the relative error e_ij of p_ij.
The sum of n terms in fp32 adds n 2^-24 of itself, and the old value two roundings; results below the
smallest normal number may be taken as 0.
"""
from __future__ import annotations

import torch

import paged_ref as ref


def logsumexps(b, causal, scale):
    """[total, heads_q] in fp32, as an attention call leaves them; rows of no sequence are NaN."""
    return ref.attention(b.q, b.k_cache, torch.nan_to_num(b.v_cache.float(), 0.0).to(b.v_cache.dtype), *b.where,
                         causal, scale, b.k_scale, None if b.v_scale is None else torch.ones_like(b.v_scale))[1].float()


def weights(b, lse, old, causal, scale, reset_new=True):
    """(weights, tolerance) [pages, heads, page] in 64 bits."""
    hk, page = b.k_cache.shape[1], b.k_cache.shape[2]
    total, hq, d = b.q.shape
    group = hq // hk
    out, tol = old.double().clone(), torch.zeros(old.shape, dtype=torch.float64, device=old.device)
    offsets, lens = b.offsets.tolist(), b.lens.tolist()
    for s, n in enumerate(lens):
        a, z = offsets[s], offsets[s + 1]
        count = z - a
        if count == 0 or n == 0:
            continue
        x = b.q[a:z].double().view(count, hk, group, d)
        k = ref.dequantise(ref.gather(b.k_cache, b.table, s, n),
                           None if b.k_scale is None else ref.gather(b.k_scale, b.table, s, n))
        z_ = torch.einsum("ihgd,jhd->hgij", x, k) * scale
        size = torch.einsum("ihgd,jhd->hgij", x.abs(), k.abs()) * abs(scale)
        l = lse[a:a + count].double().view(count, hk, group).permute(1, 2, 0)[..., None]
        p = torch.exp(z_ - l)
        e = (d + 8) * 2.0 ** -23 * size + 2.0 ** -21 * (1 + z_.abs() + l.abs())
        dead = torch.isneginf(l).expand_as(p)
        if causal:
            i = torch.arange(count, device=old.device)[:, None] + n - count
            dead = dead | (torch.arange(n, device=old.device)[None] > i)
        p = p.masked_fill(dead, 0.0)
        got = p.sum((1, 2))
        off = (p * e.masked_fill(dead, 0.0)).sum((1, 2)) + count * group * (2.0 ** -24 * got + 2.0 ** -126)
        j = torch.arange(n, device=old.device)
        where = (b.table[s, j // page].long(), slice(None), j % page)
        before = out[where].clone()
        if reset_new:
            before[max(0, n - count):] = 0
        out[where] = before + got.T
        tol[where] = off.T + 2.0 ** -22 * (before.abs() + got.T)
    return out, tol
