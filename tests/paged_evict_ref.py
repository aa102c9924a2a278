"""Eviction from a paged cache, step by step on the host: every result is exact."""
from __future__ import annotations

import math

import torch


def bits(x):
    """A tensor's bytes: comparisons that no NaN hides from."""
    return x.contiguous().view(torch.uint8)


def evict(caches, weights, table, lens, keep, recent, to_table=None):
    """(new_lens, kept, the caches behind it), on the CPU.  `caches`: tensors [pages, heads, page, ..] that
    are moved alike, `weights` among them."""
    page, heads = weights.shape[2], weights.shape[1]
    w = weights.cpu()
    old = [bits(x.cpu()).view(*x.shape[:3], -1) for x in caches]
    new = [x.clone() for x in old]
    table, lens = table.cpu(), lens.cpu().tolist()
    to = table if to_table is None else to_table.cpu()
    kept = torch.full((len(lens), heads, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pos = torch.arange(n)
        at = w[table[b, pos // page].long(), :, pos % page].tolist()
        for h in range(heads):
            if n <= keep:
                stay = list(range(n))
            else:
                def place(i):
                    return (0, 0.0, i) if math.isnan(at[i][h]) else (1, -at[i][h], i)
                stay = sorted(sorted(range(n - recent), key=place)[:keep - recent]) + list(range(n - recent, n))
            if not stay:
                continue
            kept[b, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
            s, i = torch.tensor(stay), torch.arange(len(stay))
            for x, y in zip(new, old):
                x[to[b, i // page].long(), h, i % page] = y[table[b, s // page].long(), h, s % page]
    return torch.tensor([min(n, keep) for n in lens], dtype=torch.int32), kept, new
