"""Timed cases of the paged key/value cache: writing it, reading it back, attending over it.

B sequences share caches of pages, `k_cache` and `v_cache` [pages, heads_kv, page_size, head_dim].
`page_table` [B, columns] lists each sequence's pages, `kv_lens` [B] its length in tokens with the
new ones, and `offsets` [B + 1] its rows in the packed tensors of new tokens: row i of sequence b is
the token at position kv_lens[b] - (offsets[b + 1] - offsets[b]) + i.  A float8 e4m3 cache holds
each (token, head) row divided by a power of two, which is kept in `k_scale` / `v_scale`
[pages, heads_kv, page_size].

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
          lens=1):
    """q, kv: (shortest, longest) number of new tokens and cache length of a sequence."""
    return {"name": name, "op": op, "dtype": dtype, "cache": cache, "seqs": seqs, "q_min": q[0],
            "q_max": q[1], "kv_min": kv[0], "kv_max": kv[1], "heads_q": heads_q,
            "heads_kv": heads_kv, "head_dim": head_dim, "page_size": page_size, "causal": causal,
            "lens": lens}


def listed():
    return [
        # one new token of each running sequence goes to a float8 cache: the smallest call
        _case("write-step-fp8", "write", "bf16", "fp8", 16, (1, 1), (20, 2000), 16, 8, 128, 64),
        # a batch of prompts goes to a float8 cache
        _case("write-prompts-fp8", "write", "bf16", "fp8", 9, (700, 4000), (4000, 6000), 16, 8, 128, 64),
        # odd chunks go to a 16-bit cache of short heads
        _case("write-chunks-16bit", "write", "fp16", "same", 5, (33, 2047), (2047, 5000), 16, 16, 64, 16),
        # sequences are moved off the cache: long ones, dequantised
        _case("read-long-fp8", "read", "bf16", "fp8", 4, (5000, 30000), (30000, 30001), 16, 8, 128, 64),
        # short tails of a 16-bit cache, for the dense attention of a prefix
        _case("read-short-16bit", "read", "fp16", "same", 7, (1, 900), (900, 1500), 16, 4, 64, 32),
        # one user's answer, token by token, short context
        _case("decode-one", "attend", "bf16", "same", 1, (1, 1), (777, 777), 16, 16, 128, 64),
        # a serving batch at its ordinary load, contexts of unequal length
        _case("decode-batch", "attend", "bf16", "same", 64, (1, 1), (500, 8192), 32, 8, 128, 16),
        # the same on a float8 cache with longer contexts
        _case("decode-batch-fp8", "attend", "bf16", "fp8", 40, (1, 1), (1000, 16384), 32, 8, 128, 64),
        # one very long context with few kv heads
        _case("decode-long", "attend", "fp16", "same", 1, (1, 1), (131067, 131067), 32, 4, 64, 128),
        # a few drafted tokens of each sequence are checked at once
        _case("verify-drafts", "attend", "bf16", "same", 16, (2, 8), (1000, 8192), 32, 8, 128, 64),
        # the next chunk of long prompts
        _case("chunk-long", "attend", "bf16", "same", 4, (700, 1024), (4096, 16384), 32, 8, 128, 64),
        # chunks and single tokens in one call, on a float8 cache
        _case("chunk-mixed-fp8", "attend", "fp16", "fp8", 12, (1, 600), (600, 8192), 16, 4, 128, 64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


_MOST_FLOPS = 4.0e11   # of a drawn attention: below the largest listed case's
_MOST_SCORES = 1 << 31  # padded logits of the plain form
_MOST_HELD = 1 << 29    # padded elements of a cache


def draw(rng):
    while True:
        op = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
        head_dim = rng.choice([64, 64, 128, 128, 128, 256, 32, 16])
        heads_kv = rng.choice([1, 2, 4, 8, 8, 16])
        group = rng.choice([1, 2, 3, 4, 4, 7, 8])
        cache = rng.choice(["same", "fp8"])
        page = rng.choice([8, 16, 32, 64, 64, 128, 256])
        seqs = _log_int(rng, 1, 96)
        kv_max = _log_int(rng, 30, 60000)
        kv_min = _log_int(rng, 1, kv_max)
        if op == "attend":
            q_max = 1 if rng.random() < 0.4 else _log_int(rng, 1, min(1500, kv_max))
        else:
            q_max = _log_int(rng, 1, kv_max)
        q_min = q_max if rng.random() < 0.3 else _log_int(rng, 1, q_max)
        kv_min, kv_max = max(kv_min, q_max), max(kv_max, q_max)
        case = _case("", op, rng.choice(["bf16", "fp16"]), cache, seqs, (q_min, q_max),
                     (kv_min, kv_max), heads_kv * group, heads_kv, head_dim, page,
                     rng.random() < 0.8, rng.randrange(1 << 20))
        del case["name"]
        if seqs * kv_max * heads_kv * head_dim > _MOST_HELD:
            continue
        if op == "attend" and (work(case)["flops"] > _MOST_FLOPS
                               or seqs * heads_kv * group * q_max * kv_max > _MOST_SCORES):
            continue
        return case


def _lengths(case):
    """(new tokens, cache length) of each sequence: the case's, whatever the seed of its inputs."""
    rng = random.Random(case["lens"])
    q = [_log_int(rng, case["q_min"], case["q_max"]) for _ in range(case["seqs"])]
    kv = [max(n, rng.randint(case["kv_min"], case["kv_max"])) for n in q]
    return q, kv


def work(case):
    q, kv = _lengths(case)
    hk, hq, d = case["heads_kv"], case["heads_q"], case["head_dim"]
    held = (d + 4 if case["cache"] == "fp8" else 2 * d) * hk * 2  # bytes of a cached token
    n, tables = sum(q), 4 * sum(-(-x // case["page_size"]) for x in kv) + 8 * len(q)
    if case["op"] != "attend":
        return {"bytes": n * (held + 2 * 2 * hk * d) + tables, "flops": 0}
    pairs = sum(a * c - (a * (a - 1) // 2 if case["causal"] else 0) for a, c in zip(q, kv))
    return {"bytes": sum(kv) * held + n * hq * (2 * 2 * d + 4) + tables, "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------------------- the inputs
def _scales(x):
    """2^e with the smallest e >= -126 for which a row's largest magnitude is at most 448 * 2^e."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    return ((torch.where(m == 0, torch.zeros_like(e), e) + 127) << 23).view(torch.float32)


def _quantised(x):
    x = x.float()
    s = _scales(x)
    return (x / s[..., None]).to(_FP8), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    hk, hq, d, page = case["heads_kv"], case["heads_q"], case["head_dim"], case["page_size"]
    q, kv = _lengths(case)
    per = [-(-n // page) for n in kv]
    total, columns = sum(per), max(per)
    pages = total + 3  # a few pages are free
    order = torch.randperm(pages, generator=g, device=dev)[:total].to(torch.int32)
    table = torch.full((len(q), columns), -1, dtype=torch.int32)
    at = 0
    order = order.cpu()
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    offsets = torch.tensor([0] + q).cumsum(0).to(torch.int32)
    n = sum(q)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32)

    # keys have channels of larger magnitude, values rows of unequal magnitude
    channels = torch.exp(0.5 * normal(hk, 1, d))

    def rows(gain):
        out = torch.empty((pages, hk, page, d), dtype=dtype, device=dev)
        step = max(1, (1 << 27) // (hk * page * d))
        for a in range(0, pages, step):
            m = min(step, pages - a)
            x = normal(m, hk, page, d)
            out[a:a + m] = x * (channels if gain else torch.exp(0.3 * normal(m, hk, page, 1)))
        return out

    s = {"op": case["op"], "offsets": offsets.to(dev), "kv_lens": torch.tensor(kv, dtype=torch.int32).to(dev),
         "page_table": table.to(dev), "total": n, "max_q": max(q), "max_kv": max(kv), "dtype": dtype,
         "causal": case["causal"], "sm_scale": d ** -0.5, "k_scale": None, "v_scale": None}
    if case["op"] == "write":
        held = _FP8 if case["cache"] == "fp8" else dtype
        for name in ("k", "v"):
            s[name + "_cache"] = torch.zeros((pages, hk, page, d), dtype=dtype, device=dev).to(held)
            if held == _FP8:
                s[name + "_scale"] = torch.ones((pages, hk, page), device=dev)
        # as a projection of q, k and v leaves them: one tensor, cut
        mixed = normal(n, hq + 2 * hk, d)
        mixed[:, hq:hq + hk] *= channels[:, 0]
        mixed = mixed.to(dtype)
        s["k"], s["v"] = mixed[:, hq:hq + hk], mixed[:, hq + hk:]
        return s
    for name in ("k", "v"):
        x = rows(name == "k")
        if case["cache"] == "fp8":
            held = torch.empty(x.shape, dtype=_FP8, device=dev)
            scale = torch.empty(x.shape[:3], device=dev)
            step = max(1, (1 << 27) // (hk * page * d))
            for a in range(0, pages, step):
                c, scale[a:a + step] = _quantised(x[a:a + step])
                held[a:a + step] = c
            x, s[name + "_scale"] = held, scale
        s[name + "_cache"] = x
    if case["op"] == "attend":
        s["q"] = normal(n, hq, d).to(dtype)
    return s


# ------------------------------------------------------------------------------ the plain forms
def _bytes(x):
    return x.view(torch.uint8) if x.dtype == _FP8 else x


def _places(s):
    """(page, row in the page) of every new token."""
    t = torch.arange(s["total"], device=s["offsets"].device)
    b = torch.searchsorted(s["offsets"][1:], t, right=True)
    pos = s["kv_lens"][b] - s["offsets"][b + 1] + t
    size = s["k_cache"].shape[2]
    return s["page_table"][b, pos // size].long(), pos % size


def _write(s):
    page, row = _places(s)
    for name in ("k", "v"):
        x, cache, scale = s[name], s[name + "_cache"], s[name + "_scale"]
        if scale is not None:
            x, e = _quantised(x)
            scale[page, :, row] = e
        _bytes(cache)[page, :, row] = _bytes(x)
    held = [s["k_cache"], s["v_cache"]]
    return held if s["k_scale"] is None else held + [s["k_scale"], s["v_scale"]]


def _gathered(s, name, page, row):
    """Cache rows at (page, row), in 32 bits: [..., heads_kv, head_dim]."""
    cache, scale = s[name + "_cache"], s[name + "_scale"]
    x = _bytes(cache)[page, :, row].view(cache.dtype).float()
    return x if scale is None else x * scale[page, :, row][..., None]


def _read(s):
    page, row = _places(s)
    return [_gathered(s, name, page, row).to(s["dtype"]) for name in ("k", "v")]


def _attend(s):
    dev = s["q"].device
    n, hq, d = s["q"].shape
    hk, size = s["k_cache"].shape[1:3]
    offsets, lens = s["offsets"].long(), s["kv_lens"].long()
    seqs, mq, mk = lens.numel(), s["max_q"], s["max_kv"]
    pos = torch.arange(mk, device=dev)
    page = s["page_table"][:, pos // size].long().clamp(min=0)
    row = (pos % size).expand(seqs, mk)
    k = _gathered(s, "k", page, row).permute(0, 2, 3, 1)      # [B, Hkv, D, keys]
    v = _gathered(s, "v", page, row).transpose(1, 2)          # [B, Hkv, keys, D]
    count = offsets[1:] - offsets[:-1]
    i = torch.arange(mq, device=dev)
    at = (offsets[:-1, None] + i).clamp(max=n - 1)
    x = s["q"].float()[at].view(seqs, mq, hk, hq // hk, d).transpose(1, 2)
    logits = torch.matmul(x.reshape(seqs, hk, -1, d), k).view(seqs, hk, mq, hq // hk, mk)
    logits *= s["sm_scale"]
    last = lens - 1 if not s["causal"] else lens - count
    last = last[:, None] + (i if s["causal"] else 0 * i)      # the last key of each row
    hidden = (pos > torch.minimum(last, lens[:, None] - 1)[..., None])[:, None, :, None]
    logits.masked_fill_(hidden, float("-inf"))
    most = logits.amax(-1, keepdim=True)
    most = torch.where(most == float("-inf"), torch.zeros_like(most), most)
    p = logits.sub_(most).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs, hk, -1, mk), v).view(seqs, hk, mq, hq // hk, d)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    lse = (most + total.log())[..., 0]
    t = torch.arange(n, device=dev)
    b = torch.searchsorted(offsets[1:], t, right=True)
    i = t - offsets[b]
    return [out[b, :, i].reshape(n, hq, d).to(s["dtype"]), lse[b, :, i].reshape(n, hq)]


def run(s):
    if own:
        import flash_attention_forward as fa

        where = (s["page_table"], s["offsets"], s["kv_lens"])
        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if s["op"] == "write":
            fa.paged_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], *where, **scales)
            held = [s["k_cache"], s["v_cache"]]
            return held if s["k_scale"] is None else held + [s["k_scale"], s["v_scale"]]
        if s["op"] == "read":
            return list(fa.paged_cache_read(s["k_cache"], s["v_cache"], *where, s["total"],
                                            dtype=s["dtype"], **scales))
        return list(fa.paged_attention(s["q"], s["k_cache"], s["v_cache"], *where, s["causal"],
                                       s["sm_scale"], max_q_len=s["max_q"], return_lse=True,
                                       **scales))
    return {"write": _write, "read": _read, "attend": _attend}[s["op"]](s)


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definition, sequence by sequence, in 64 bits.  A float8 cache's rows are None: what a
    rounding to 4 bits gives has no 64-bit value; their scales are powers of two."""
    s = prepare(case, seed)
    q, kv = _lengths(case)
    page = case["page_size"]
    group = case["heads_q"] // case["heads_kv"]

    def held(name, b, first, last):
        """Rows first .. last of sequence b, [rows, heads_kv, head_dim]."""
        pages = s["page_table"][b, :-(-last // page)].long()
        x = s[name + "_cache"][pages].double().transpose(1, 2).flatten(0, 1)
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][pages].double().transpose(1, 2).flatten(0, 1)[..., None]
        return x[first:last]

    if case["op"] == "read":
        return [torch.cat([held(name, b, kv[b] - q[b], kv[b]) for b in range(len(q))])
                for name in ("k", "v")]
    if case["op"] == "write":
        out, scales = [], []
        for name in ("k", "v"):
            cache = s[name + "_cache"].double()
            scale = s[name + "_scale"]
            at = 0
            for b in range(len(q)):
                pos = torch.arange(kv[b] - q[b], kv[b], device=cache.device)
                pages, rows = s["page_table"][b, pos // page].long(), pos % page
                x = s[name][at:at + q[b]].double()
                at += q[b]
                cache[pages, :, rows] = x
                if scale is not None:
                    top = x.abs().amax(-1)
                    least = torch.exp2(torch.floor(torch.log2(top / 448)) - 1)  # doubled until enough
                    for _ in range(4):
                        least = torch.where(448 * least < top, 2 * least, least)
                    scale[pages, :, rows] = torch.where(top == 0, 1.0, least).float()
            out.append(None if scale is not None else cache)
            scales.append(scale.double() if scale is not None else None)
        return out if scales[0] is None else out + scales
    outs, sums = [], []
    at = 0
    for b in range(len(q)):
        k, v = (held(name, b, 0, kv[b]).transpose(0, 1) for name in ("k", "v"))
        x = s["q"][at:at + q[b]].double().view(q[b], -1, group, case["head_dim"]).permute(1, 2, 0, 3)
        at += q[b]
        o = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        m = torch.empty(x.shape[:3], dtype=torch.float64, device=x.device)
        hidden = None
        if case["causal"]:
            hidden = torch.ones((q[b], kv[b]), dtype=torch.bool, device=x.device).triu(kv[b] - q[b] + 1)
        for h in range(k.shape[0]):
            z = torch.einsum("gid,jd->gij", x[h], k[h]) * s["sm_scale"]
            if hidden is not None:
                z.masked_fill_(hidden, float("-inf"))
            m[h] = torch.logsumexp(z, -1)
            o[h] = torch.einsum("gij,jd->gid", torch.exp(z - m[h][..., None]), v[h])
        outs.append(o.permute(2, 0, 1, 3).flatten(1, 2))
        sums.append(m.permute(2, 0, 1).flatten(1, 2))
    return [torch.cat(outs), torch.cat(sums)]
