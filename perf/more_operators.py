"""Timed cases of three operators around the paged key/value cache: attention of a batch that shares
long prefixes, the attention weight that each cached token received, and eviction by that weight.

Sequences share caches of pages, `k_cache` and `v_cache` [pages, heads_kv, page_size, head_dim].
`page_table` [B, columns] lists each sequence's pages, `kv_lens` [B] its length in tokens, and
`offsets` [B + 1] its rows in the packed tensors of new tokens.  A float8 e4m3 cache holds each
(token, head) row divided by a power of two, kept in `k_scale` / `v_scale` [pages, heads_kv,
page_size].  A shared prefix is held once: `prefix_table`, `prefix_lens` list its pages and length,
and `prefix_offsets` the packed rows that attend to it before their sequence's own tokens.  `weights`
[pages, heads_kv, page_size] float32 holds the attention weight of each (token, kv head).

With `own` false, `run` computes the operators from elementary torch operations in 32 bits; with
`own` true it calls the framework's kernels.
"""
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_FP8 = torch.float8_e4m3fn


# ------------------------------------------------------------------------------------ the cases
def _case(name, op, dtype, cache, seqs, q, kv, heads_q, heads_kv, head_dim, page_size, causal=True,
          groups=0, prefix=(0, 0), keep=0, recent=0, in_place=True, lens=1):
    """q, kv: (shortest, longest) number of new tokens and cache length of a sequence; prefix: of a
    shared prefix; keep, recent: tokens that an eviction leaves, and the last ones that it spares."""
    return {"name": name, "op": op, "dtype": dtype, "cache": cache, "seqs": seqs, "q_min": q[0],
            "q_max": q[1], "kv_min": kv[0], "kv_max": kv[1], "heads_q": heads_q,
            "heads_kv": heads_kv, "head_dim": head_dim, "page_size": page_size, "causal": causal,
            "groups": groups, "prefix_min": prefix[0], "prefix_max": prefix[1], "keep": keep,
            "recent": recent, "in_place": in_place, "lens": lens}


def listed():
    return [
        # a few samples of one prompt, decoded together: the smallest call
        _case("prefix-few", "prefix", "bf16", "same", 4, (1, 1), (20, 300), 16, 16, 128, 64,
              groups=1, prefix=(1000, 1000)),
        # a serving batch behind one long system prompt
        _case("prefix-batch", "prefix", "bf16", "same", 64, (1, 1), (100, 2000), 32, 8, 128, 16,
              groups=1, prefix=(8191, 8191)),
        # drafted tokens of users of three documents, on a float8 cache
        _case("prefix-drafts-fp8", "prefix", "bf16", "fp8", 40, (1, 5), (50, 4000), 32, 8, 128, 64,
              groups=3, prefix=(4000, 20000)),
        # questions (many tokens each) about one document, short heads
        _case("prefix-chunks", "prefix", "fp16", "same", 6, (200, 700), (700, 1500), 16, 4, 64, 32,
              groups=1, prefix=(6001, 6001)),
        # a decoding step of short sequences in a float8 cache
        _case("weights-step-fp8", "weights", "bf16", "fp8", 16, (1, 1), (100, 2000), 16, 8, 128, 64),
        # a decoding step of a serving batch
        _case("weights-batch", "weights", "bf16", "same", 64, (1, 1), (500, 8192), 32, 8, 128, 16),
        # prompts, whole: a cache is cut to size after them
        _case("weights-prompts", "weights", "bf16", "same", 5, (700, 3500), (1, 1), 32, 8, 128, 64),
        # the next chunk of long prompts, float8
        _case("weights-chunks-fp8", "weights", "fp16", "fp8", 4, (300, 1024), (4096, 16384), 16, 4, 64, 128),
        # running sequences that grew by a page over their budget
        _case("evict-step", "evict", "bf16", "same", 16, (0, 0), (576, 576), 16, 8, 128, 64, keep=512,
              recent=64),
        # a serving batch of unequal lengths on a float8 cache, some below the budget
        _case("evict-batch-fp8", "evict", "bf16", "fp8", 48, (0, 0), (800, 6000), 16, 8, 128, 64,
              keep=1024, recent=128),
        # prompts cut to a budget, into pages of their own, which frees theirs
        _case("evict-prompts", "evict", "fp16", "same", 7, (0, 0), (2500, 20000), 16, 16, 64, 16,
              keep=2048, recent=256, in_place=False),
        # one very long context with few kv heads
        _case("evict-long", "evict", "bf16", "same", 1, (0, 0), (131067, 131067), 32, 4, 128, 128,
              keep=40000, recent=1000),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


_MOST_FLOPS = 2.0e11    # of a drawn case: below the largest listed one's
_MOST_SCORES = 1 << 30  # padded logits of the plain form
_MOST_HELD = 1 << 28    # padded elements of a cache


def draw(rng):
    while True:
        op = rng.choice(["prefix", "weights", "evict"])
        head_dim = rng.choice([64, 64, 128, 128, 128, 256, 32, 16])
        heads_kv = rng.choice([1, 2, 4, 8, 8, 16])
        group = rng.choice([1, 2, 3, 4, 4, 7, 8])
        seqs = _log_int(rng, 1, 96)
        page = rng.choice([8, 16, 32, 64, 64, 128, 256])
        common = dict(lens=rng.randrange(1 << 20))
        types = rng.choice(["bf16", "fp16"]), rng.choice(["same", "fp8"])
        kv_max = _log_int(rng, 30, 60000)
        if op == "evict":
            kv_min = _log_int(rng, 1, kv_max)
            common["keep"] = _log_int(rng, 16, max(16, kv_max))
            common["recent"] = rng.randrange(common["keep"] + 1)
            common["in_place"] = rng.random() < 0.6
            q_min = q_max = 0
        else:
            q_max = 1 if rng.random() < 0.4 else _log_int(rng, 1, min(1500, kv_max))
            q_min = q_max if rng.random() < 0.3 else _log_int(rng, 1, q_max)
            kv_min, kv_max = max(_log_int(rng, 1, kv_max), q_max), max(kv_max, q_max)
            common["causal"] = rng.random() < 0.8
            if op == "prefix":
                kv_max = max(q_max, kv_max // 8)
                kv_min = min(kv_min, kv_max)
                common["groups"] = rng.randint(1, min(4, seqs))
                top = _log_int(rng, 30, 60000)
                common["prefix"] = _log_int(rng, 1, top), top
        case = _case("", op, *types, seqs, (q_min, q_max), (kv_min, kv_max), heads_kv * group, heads_kv,
                     head_dim, page, **common)
        del case["name"]
        held = seqs * kv_max + case["groups"] * case["prefix_max"]
        if held * heads_kv * head_dim > _MOST_HELD:
            continue
        rows = heads_kv * group * q_max * seqs
        if rows * (kv_max + case["prefix_max"] * max(1, case["groups"])) > _MOST_SCORES:
            continue
        if work(case)["flops"] > _MOST_FLOPS:
            continue
        return case


def _lengths(case):
    """(new tokens, cache length) of each sequence, and each prefix's (sequences, length): the case's,
    whatever the seed of its inputs."""
    rng = random.Random(case["lens"])
    q = [_log_int(rng, case["q_min"], case["q_max"]) if case["q_max"] else 0 for _ in range(case["seqs"])]
    kv = [max(n, rng.randint(case["kv_min"], case["kv_max"])) for n in q]
    g = case["groups"]
    cuts = [0] + sorted(rng.sample(range(1, case["seqs"]), g - 1)) + [case["seqs"]] if g else [0]
    prefix = [rng.randint(case["prefix_min"], case["prefix_max"]) for _ in range(g)]
    return q, kv, [b - a for a, b in zip(cuts, cuts[1:])], prefix


def work(case):
    q, kv, members, prefix = _lengths(case)
    hk, hq, d = case["heads_kv"], case["heads_q"], case["head_dim"]
    row = (d + 4 if case["cache"] == "fp8" else 2 * d) * hk  # bytes of a cached token's keys
    n, page = sum(q), case["page_size"]
    tables = 4 * sum(-(-x // page) for x in kv + prefix) + 8 * len(q)
    pairs = sum(a * c - (a * (a - 1) // 2 if case["causal"] else 0) for a, c in zip(q, kv))
    if case["op"] == "prefix":
        at = 0
        for m, x in zip(members, prefix):
            pairs += sum(q[at:at + m]) * x
            at += m
        return {"bytes": 2 * row * (sum(kv) + sum(prefix)) + n * hq * (4 * d + 4) + tables,
                "flops": 4 * d * hq * pairs}
    if case["op"] == "weights":
        return {"bytes": (row + 8 * hk) * sum(kv) + n * hq * (2 * d + 4) + tables, "flops": 2 * d * hq * pairs}
    keep = case["keep"]
    cut = [x for x in kv if x > keep or not case["in_place"]]
    kept = sum(min(x, keep) for x in cut)
    return {"bytes": 4 * hk * sum(cut) + 2 * kept * (2 * row + 4 * hk) + 4 * hk * keep * len(kv) + tables,
            "flops": 0}


# ----------------------------------------------------------------------------------- the inputs
def _quantised(x):
    """Codes, and 2^e with the smallest e >= -126 for which a row's largest magnitude is at most
    448 * 2^e."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    s = ((torch.where(m == 0, torch.zeros_like(e), e) + 127) << 23).view(torch.float32)
    return (x / s[..., None]).to(_FP8), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    hk, hq, d, page = case["heads_kv"], case["heads_q"], case["head_dim"], case["page_size"]
    q, kv, members, prefix = _lengths(case)
    keep = case["keep"]
    lists = [-(-x // page) for x in kv + prefix]
    if case["op"] == "evict" and not case["in_place"]:
        lists += [-(-min(x, keep) // page) for x in kv]
    total = sum(lists)
    pages = total + 3  # a few pages are free
    order = torch.randperm(pages, generator=g, device=dev)[:total].to(torch.int32).cpu()

    def tables(per):
        nonlocal at
        table = torch.full((len(per), max(per)), -1, dtype=torch.int32)
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        return table.to(dev)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32).to(dev)

    def sums(x):
        return torch.tensor([0] + x).cumsum(0).to(torch.int32).to(dev)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32)

    at, n = 0, sum(q)
    s = {"op": case["op"], "dtype": dtype, "causal": case["causal"], "sm_scale": d ** -0.5, "total": n,
         "page_table": tables(lists[:len(kv)]), "offsets": sums(q), "kv_lens": ints(kv), "max_q": max(q),
         "max_kv": max(kv), "k_scale": None, "v_scale": None, "keep": keep, "recent": case["recent"],
         "to_table": None}
    if prefix:
        s["prefix_table"] = tables(lists[len(kv):len(kv) + len(prefix)])
        rows, b = [], 0
        for m in members:
            rows.append(sum(q[b:b + m]))
            b += m
        s |= {"prefix_offsets": sums(rows), "prefix_lens": ints(prefix), "max_rows": max(rows),
              "max_prefix": max(prefix)}
    if len(lists) > len(kv) + len(prefix):
        s["to_table"] = tables(lists[len(kv):])

    # keys have channels of larger magnitude, values rows of unequal magnitude
    channels = torch.exp(0.5 * normal(hk, 1, d))
    step = max(1, (1 << 27) // (hk * page * d))
    for name in ("k", "v"):
        held = torch.empty((pages, hk, page, d), dtype=_FP8 if case["cache"] == "fp8" else dtype, device=dev)
        scale = torch.ones((pages, hk, page), device=dev)
        for a in range(0, pages, step):
            m = min(step, pages - a)
            x = normal(m, hk, page, d)
            x = (x * (channels if name == "k" else torch.exp(0.3 * normal(m, hk, page, 1)))).to(dtype)
            if case["cache"] == "fp8":
                x, scale[a:a + m] = _quantised(x)
            held[a:a + m] = x
        s[name + "_cache"] = held
        if case["cache"] == "fp8":
            s[name + "_scale"] = scale
    if case["op"] != "evict":
        s["q"] = normal(n, hq, d).to(dtype)
    if case["op"] == "weights":
        # what the steps before left, and the sums of the attention call that these rows went through
        s["weights"] = torch.exp(normal(pages, hk, page) - 3)
        s["lse"] = _lse(s)
    if case["op"] == "evict":
        # a few tokens hold most of the weight; some never got any
        w = torch.exp(2.5 * normal(pages, hk, page) - 3)
        s["weights"] = torch.where(w < 1e-3, torch.zeros_like(w), w)
        # (an eviction reorders them: the next pass has to find them as they were)
        s["counted"] = s["weights"].clone()
    return s


# ------------------------------------------------------------------------------ the plain forms
def _bytes(x):
    return x.view(torch.uint8) if x.dtype == _FP8 else x


def _rows_of(s, name, table, mk):
    """The first mk tokens of each row of `table`, in 32 bits: [B, mk, heads_kv, head_dim]."""
    cache, scale = s[name + "_cache"], s[name + "_scale"]
    pos = torch.arange(mk, device=cache.device)
    size = cache.shape[2]
    page = table[:, pos // size].long().clamp(min=0)
    row = (pos % size).expand_as(page)
    x = _bytes(cache)[page, :, row].view(cache.dtype).float()
    return x if scale is None else x * scale[page, :, row][..., None]


def _logits(s, table, offsets, lens, causal, mq, mk):
    """Masked logits [B, heads_kv, mq, group, mk] of each row's packed queries over its tokens, and
    the (row of the table, place in it) of each packed query."""
    q = s["q"]
    n, hq, d = q.shape
    k = _rows_of(s, "k", table, mk).permute(0, 2, 3, 1)       # [B, Hkv, D, keys]
    seqs, hk = k.shape[:2]
    offsets, lens = offsets.long(), lens.long()
    i = torch.arange(mq, device=q.device)
    pos = torch.arange(mk, device=q.device)
    at = (offsets[:-1, None] + i).clamp(max=n - 1)
    x = q.float()[at].view(seqs, mq, hk, hq // hk, d).transpose(1, 2)
    z = torch.matmul(x.reshape(seqs, hk, -1, d), k).view(seqs, hk, mq, hq // hk, mk).mul_(s["sm_scale"])
    count = offsets[1:] - offsets[:-1]
    last = (lens - count)[:, None] + i if causal else (lens - 1)[:, None].expand(seqs, mq)
    last = torch.minimum(last, (lens - 1)[:, None])           # the last key of each row
    z.masked_fill_((pos > last[..., None])[:, None, :, None], float("-inf"))
    t = torch.arange(n, device=q.device)
    b = torch.searchsorted(offsets[1:], t, right=True)
    return z, b, t - offsets[b], i[None] < count[:, None]


def _lse(s):
    z, b, i, _ = _logits(s, s["page_table"], s["offsets"], s["kv_lens"], s["causal"], s["max_q"], s["max_kv"])
    return torch.logsumexp(z, -1)[b, :, i].reshape(s["q"].shape[:2])


def _parts(s, table, offsets, lens, causal, mq, mk):
    """(largest logit, sum, sum of values) of each packed query over its row of `table`."""
    z, b, i, _ = _logits(s, table, offsets, lens, causal, mq, mk)
    most = z.amax(-1, keepdim=True)
    most = torch.where(most == float("-inf"), torch.zeros_like(most), most)
    p = z.sub_(most).exp_()
    v = _rows_of(s, "v", table, mk).transpose(1, 2)
    o = torch.matmul(p.flatten(2, 3), v).view(*p.shape[:-1], v.shape[-1])
    shape = s["q"].shape[:2]
    return (most[..., 0][b, :, i].reshape(shape), p.sum(-1)[b, :, i].reshape(shape),
            o[b, :, i].reshape(s["q"].shape))


def _prefix(s):
    m1, l1, o1 = _parts(s, s["prefix_table"], s["prefix_offsets"], s["prefix_lens"], False, s["max_rows"],
                        s["max_prefix"])
    m2, l2, o2 = _parts(s, s["page_table"], s["offsets"], s["kv_lens"], s["causal"], s["max_q"], s["max_kv"])
    m = torch.maximum(m1, m2)
    a, b = torch.exp(m1 - m), torch.exp(m2 - m)
    total = l1 * a + l2 * b
    out = (o1 * a[..., None] + o2 * b[..., None]) / total[..., None]
    return [out.to(s["dtype"]), m + total.log()]


def _weights(s):
    z, _, _, live = _logits(s, s["page_table"], s["offsets"], s["kv_lens"], s["causal"], s["max_q"], s["max_kv"])
    seqs, hk, mq, group, mk = z.shape
    at = (s["offsets"][:-1, None].long() + torch.arange(mq, device=z.device)).clamp(max=s["total"] - 1)
    lse = s["lse"][at].view(seqs, mq, hk, group).transpose(1, 2)
    p = z.sub_(lse[..., None]).exp_().masked_fill_(~live[:, None, :, None, None], 0.0)
    got = p.sum((2, 3)).transpose(1, 2)                       # [B, keys, Hkv]
    w, size = s["weights"], s["k_cache"].shape[2]
    pos = torch.arange(mk, device=z.device)
    page, row = s["page_table"][:, pos // size].long(), (pos % size).expand(seqs, mk)
    lens = s["kv_lens"][:, None]
    new = pos >= lens - (s["offsets"][1:] - s["offsets"][:-1])[:, None]
    got = got + torch.where(new[..., None], torch.zeros_like(got), w[page.clamp(min=0), :, row])
    here = pos < lens
    w[page[here], :, row[here]] = got[here]
    return w


def _evict(s):
    lens, keep, recent = s["kv_lens"].long(), s["keep"], s["recent"]
    dev, size, mk = lens.device, s["k_cache"].shape[2], s["max_kv"]
    pos = torch.arange(mk, device=dev)
    page, row = s["page_table"][:, pos // size].long().clamp(min=0), (pos % size).expand(lens.numel(), mk)
    w = s["weights"][page, :, row].transpose(1, 2)            # [B, Hkv, keys]
    here = (pos < lens[:, None])[:, None]
    spared = (pos >= lens[:, None] - recent)[:, None] | (lens <= keep)[:, None, None]
    rank = torch.where(spared, torch.full_like(w, float("inf")), w).masked_fill(~here, float("-inf"))
    kept = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :keep]
    new = torch.minimum(lens, torch.full_like(lens, keep))
    i = torch.arange(kept.shape[-1], device=dev)
    live = (i < new[:, None])[:, None].expand_as(kept)
    kept = torch.sort(kept.masked_fill(~live, mk), dim=-1)[0]
    to = s["page_table"] if s["to_table"] is None else s["to_table"]
    b, h, r = live.nonzero(as_tuple=True)
    p = kept[b, h, r]
    from_page, from_row = s["page_table"][b, p // size].long(), p % size
    to_page, to_row = to[b, r // size].long(), r % size
    held = [s["k_cache"], s["v_cache"], s["weights"]]
    if s["k_scale"] is not None:
        held += [s["k_scale"], s["v_scale"]]
    for x in held:
        _bytes(x)[to_page, h, to_row] = _bytes(x)[from_page, h, from_row]
    out = torch.full((*kept.shape[:2], keep), -1, dtype=torch.int32, device=dev)
    out[..., :kept.shape[-1]] = kept.masked_fill(~live, -1)
    return [new.to(torch.int32), out] + held


def run(s):
    if s["op"] == "evict":
        s["weights"].copy_(s["counted"])
    if own:
        import flash_attention_forward as fa

        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if s["op"] == "prefix":
            return list(fa.paged_prefix_attention(
                s["q"], s["k_cache"], s["v_cache"], s["prefix_table"], s["prefix_offsets"], s["prefix_lens"],
                s["page_table"], s["offsets"], s["kv_lens"], s["causal"], s["sm_scale"], max_q_len=s["max_q"],
                max_prefix_q_len=s["max_rows"], return_lse=True, **scales))
        if s["op"] == "weights":
            fa.paged_attention_weights(s["q"], s["lse"], s["k_cache"], s["page_table"], s["offsets"],
                                       s["kv_lens"], s["weights"], s["causal"], s["sm_scale"],
                                       k_scale=s["k_scale"], max_q_len=s["max_q"])
            return s["weights"]
        new, kept = fa.paged_cache_evict(s["k_cache"], s["v_cache"], s["weights"], s["page_table"],
                                         s["kv_lens"], s["keep"], s["recent"], to_table=s["to_table"],
                                         return_kept=True, **scales)
        held = [s["k_cache"], s["v_cache"], s["weights"]]
        return [new, kept] + held + ([s["k_scale"], s["v_scale"]] if s["k_scale"] is not None else [])
    return {"prefix": _prefix, "weights": _weights, "evict": _evict}[s["op"]](s)


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions, sequence by sequence, in 64 bits."""
    s = prepare(case, seed)
    q, kv, members, prefix = _lengths(case)
    page, hk, d = case["page_size"], case["heads_kv"], case["head_dim"]
    group = case["heads_q"] // hk

    def held(name, table, b, n):
        """The first n tokens of a row of a table, [heads_kv, n, head_dim]."""
        pages = table[b, :-(-n // page)].long()
        x = s[name + "_cache"][pages].double().transpose(1, 2).flatten(0, 1)
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][pages].double().transpose(1, 2).flatten(0, 1)[..., None]
        return x[:n].transpose(0, 1)

    def hidden(b):
        if not case["causal"]:
            return None
        return torch.ones((q[b], kv[b]), dtype=torch.bool, device="cuda").triu(kv[b] - q[b] + 1)

    if case["op"] == "evict":
        new = [min(x, case["keep"]) for x in kv]
        kept = torch.full((len(kv), hk, case["keep"]), -1, dtype=torch.int32)
        names = ["k_cache", "v_cache", "weights"] + (["k_scale", "v_scale"] if s["k_scale"] is not None else [])
        after = [s[x].double() for x in names]
        to = s["page_table"] if s["to_table"] is None else s["to_table"]
        for b, x in enumerate(kv):
            pages = s["page_table"][b, :-(-x // page)].long()
            w = s["weights"][pages].transpose(1, 2).flatten(0, 1)[:x].cpu().double()
            for h in range(hk):
                old = x - case["recent"]
                if x <= case["keep"]:
                    stay = torch.arange(x)
                else:
                    order = sorted(range(old), key=list(zip((-w[:old, h]).tolist(), range(old))).__getitem__)
                    stay = torch.tensor(sorted(order[:case["keep"] - case["recent"]]) + list(range(old, x)))
                kept[b, h, :new[b]] = stay
                if new[b] == 0:
                    continue
                src, i = stay.cuda(), torch.arange(new[b], device="cuda")
                for y in after:
                    y[to[b, i // page].long(), h, i % page] = y[s["page_table"][b, src // page].long(), h, src % page]
        return [torch.tensor(new, dtype=torch.int32), kept] + after

    if case["op"] == "weights":
        out, at = s["weights"].double(), 0
        for b in range(len(q)):
            k = held("k", s["page_table"], b, kv[b])
            x = s["q"][at:at + q[b]].double().view(q[b], hk, group, d).permute(1, 2, 0, 3)
            lse = s["lse"][at:at + q[b]].double().view(q[b], hk, group).permute(1, 2, 0)
            at += q[b]
            mask, sums = hidden(b), torch.zeros((hk, kv[b]), dtype=torch.float64, device="cuda")
            for h in range(hk):
                for j in range(group):
                    p = torch.exp(x[h, j] @ k[h].T * s["sm_scale"] - lse[h, j][:, None])
                    sums[h] += (p if mask is None else p.masked_fill(mask, 0.0)).sum(0)
            i = torch.arange(kv[b], device="cuda")
            where = (s["page_table"][b, i // page].long(), slice(None), i % page)
            old = out[where].clone()
            old[kv[b] - q[b]:] = 0
            out[where] = old + sums.T
        return out

    outs, sums, at, b = [], [], 0, 0
    for grp, m in enumerate(members):
        pk, pv = (held(x, s["prefix_table"], grp, prefix[grp]) for x in ("k", "v"))
        for b in range(b, b + m):
            k, v = (held(x, s["page_table"], b, kv[b]) for x in ("k", "v"))
            x = s["q"][at:at + q[b]].double().view(q[b], hk, group, d).permute(1, 2, 0, 3)
            at += q[b]
            o = torch.empty(x.shape, dtype=torch.float64, device="cuda")
            lse = torch.empty(x.shape[:3], dtype=torch.float64, device="cuda")
            mask = hidden(b)
            for h in range(hk):
                z = x[h] @ k[h].T * s["sm_scale"]
                if mask is not None:
                    z.masked_fill_(mask, float("-inf"))
                z = torch.cat([x[h] @ pk[h].T * s["sm_scale"], z], -1)
                lse[h] = torch.logsumexp(z, -1)
                o[h] = torch.exp(z - lse[h][..., None]) @ torch.cat([pv[h], v[h]])
            outs.append(o.permute(2, 0, 1, 3).flatten(1, 2))
            sums.append(lse.permute(2, 0, 1).flatten(1, 2))
        b += 1
    return [torch.cat(outs), torch.cat(sums)]
