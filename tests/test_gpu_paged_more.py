"""Prefix attention, attention weights and eviction: a run of them together, on streams, captured, as
registered operators, beyond 32-bit offsets, and their bounded waits (B200)."""
from __future__ import annotations

import ctypes
import json
import os
import subprocess
import sys

import pytest
import torch

import flash_attention_forward as fam
import paged_evict_ref as ref_e
import paged_prefix_ref as pre
import paged_ref as ref
import paged_weights_ref as ref_w
from conftest import REPO
from flash_attn_npu_b200 import build, ops, paged, torch_op  # noqa: F401  (registers the operators)

pytestmark = pytest.mark.gpu
OPS = torch.ops.flash_attn_b200
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def binding(native_lib):
    build.build_binding()


class Server:
    """Sequences behind one prefix, that decode, count weights and are cut to a budget."""

    def __init__(self, device, fp8, seed=0, seqs=5, prefix=150, page=16, heads_q=8, heads_kv=2, dim=64):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dev, self.page, self.dim, self.hq, self.hk = g, device, page, dim, heads_q, heads_kv
        per, shared = 12, -(-prefix // page)
        pages = seqs * per + shared + 3
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = order[:seqs * per].view(seqs, per).to(device)
        self.prefix = (order[seqs * per:seqs * per + shared].view(1, -1).to(device),
                       torch.tensor([0, 0], dtype=torch.int32, device=device),
                       torch.tensor([prefix], dtype=torch.int32, device=device))
        cache = fam.paged_cache_empty(pages, page, heads_kv, dim, ref.FP8 if fp8 else BF16, device)
        for x in cache:
            if x is not None:
                x.view(torch.uint8).fill_(0x7f)  # NaN until it is written
        self.k, self.v, ks, vs = cache
        self.scales = {"k_scale": ks, "v_scale": vs}
        self.w = torch.full((pages, heads_kv, page), float("nan"), device=device)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=device)
        k, v = self.rows(prefix, heads_kv), self.rows(prefix, heads_kv)
        at = torch.tensor([0, prefix], dtype=torch.int32, device=device)
        fam.paged_cache_write(k, v, self.k, self.v, self.prefix[0], at, self.prefix[2], **self.scales)
        self.w[self.prefix[0].long()] = 0

    def rows(self, n, heads):
        return torch.randn(n, heads, self.dim, generator=self.g).to(BF16).to(self.dev)

    def step(self, counts):
        """New tokens of each sequence: written, attended with, counted.  Returns what the checks need."""
        n = sum(counts)
        offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(self.dev)
        self.lens += offsets.diff()
        self.prefix[1][1] = n
        fam.paged_cache_write(self.rows(n, self.hk), self.rows(n, self.hk), self.k, self.v, self.table, offsets,
                              self.lens, **self.scales)
        q = self.rows(n, self.hq)
        out, lse = fam.paged_prefix_attention(q, self.k, self.v, *self.prefix, self.table, offsets, self.lens, True, 0.125,
                                              max_q_len=max(counts), return_lse=True, **self.scales)
        before = self.w.clone()
        more = dict(k_scale=self.scales["k_scale"], max_q_len=max(counts))
        fam.paged_attention_weights(q, lse, self.k, self.table, offsets, self.lens, self.w, True, 0.125, **more)
        fam.paged_attention_weights(q, lse, self.k, *self.prefix, self.w, False, 0.125, reset_new=False,
                                    k_scale=self.scales["k_scale"])
        return q, offsets, out, lse, before

    def view(self, q, offsets):
        """What the references look at."""
        class View:
            pass
        x = View()
        x.q, x.k_cache, x.v_cache, x.offsets, x.lens, x.table = q, self.k, self.v, offsets, self.lens, self.table
        x.prefix_table, x.prefix_offsets, x.prefix_lens = self.prefix
        x.k_scale, x.v_scale = self.scales["k_scale"], self.scales["v_scale"]
        return x


@pytest.mark.parametrize("fp8", [False, True])
def test_run_together(fp8, cuda_device):
    """Prompts, tokens, counting and eviction in turns: every step against 64 bits, every move by its bytes."""
    s = Server(cuda_device, fp8)
    for turn, counts in enumerate([[30, 1, 77, 120, 9], [1] * 5, [3, 1, 0, 2, 5], [1] * 5, [40, 2, 1, 1, 60]]):
        q, offsets, out, lse, before = s.step(counts)
        x = s.view(q, offsets)
        want, want_lse, tol, tol_lse = pre.attention(x, True, 0.125)
        assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= tol_lse).all()
        b = s.view(q, offsets)
        w1, t1 = ref_w.weights(b, lse, before, True, 0.125)
        b.table, b.offsets, b.lens = s.prefix
        w2, t2 = ref_w.weights(b, lse, w1.float(), False, 0.125, reset_new=False)
        live = ~torch.isnan(w2)
        assert torch.equal(live, ~torch.isnan(s.w))
        assert ((s.w.double() - w2).abs() <= t1 + t2 + 2.0 ** -24 * w2.abs())[live].all()
        if turn % 2 == 0:
            held = [s.k, s.v, s.w] + ([s.scales["k_scale"], s.scales["v_scale"]] if fp8 else [])
            lens, kept, moved = ref_e.evict(held, s.w, s.table, s.lens, 64, 8)
            s.lens, got = fam.paged_cache_evict(s.k, s.v, s.w, s.table, s.lens, 64, 8, return_kept=True, **s.scales)
            assert torch.equal(s.lens.cpu(), lens) and torch.equal(got.cpu(), kept)
            for a, z in zip(held, moved):
                assert torch.equal(ref_e.bits(a.cpu()).view(z.shape), z)
    ops.check_device_status(cuda_device)


@pytest.mark.parametrize("fp8", [False, True])
def test_captured_run_on_another_stream(fp8, cuda_device):
    """The same bits from calls one by one and from a replayed graph, on a stream of its own."""
    a, b = Server(cuda_device, fp8, seed=3), Server(cuda_device, fp8, seed=3)
    for s in (a, b):
        s.step([30, 1, 77, 120, 9])
    q = a.rows(5, a.hq)
    offsets = torch.arange(6, dtype=torch.int32, device=cuda_device)

    def turn(s):
        s.prefix[1].copy_(torch.stack([offsets[0], offsets[5]]))
        out, lse = fam.paged_prefix_attention(q, s.k, s.v, *s.prefix, s.table, offsets, s.lens, True, 0.125, max_q_len=1,
                                              max_prefix_q_len=5, return_lse=True, **s.scales)
        fam.paged_attention_weights(q, lse, s.k, s.table, offsets, s.lens, s.w, True, 0.125, max_q_len=1,
                                    k_scale=s.scales["k_scale"], reset_new=False)
        return out, lse, *fam.paged_cache_evict(s.k, s.v, s.w, s.table, s.lens, 50, 5, return_kept=True, **s.scales)

    torch.cuda.synchronize()
    stream = torch.cuda.Stream(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = turn(b)
    with torch.cuda.stream(stream):
        graph.replay()
    want = turn(a)
    torch.cuda.synchronize()
    for x, y in zip((*got, b.w, b.k.view(torch.uint8), b.v.view(torch.uint8)),
                    (*want, a.w, a.k.view(torch.uint8), a.v.view(torch.uint8))):
        assert torch.equal(x.nan_to_num(0.0) if x.is_floating_point() else x,
                           y.nan_to_num(0.0) if y.is_floating_point() else y)


def test_calls_on_two_streams_at_once(cuda_device):
    """Workspaces of calls that run side by side are apart."""
    work = []
    for t in range(2):
        x = pre.PrefixBatch([1] * 30, [40 * i + 1 for i in range(30)], [6000, 2000], [20, 10], heads_q=16, heads_kv=4,
                            head_dim=64, device=cuda_device, seed=t)
        p = ref.Batch([400], [3000], heads_q=8, heads_kv=1, head_dim=64, device=cuda_device, seed=t)
        work.append((x, p, ref_w.logsumexps(p, True, 0.1)))

    def calls(x, p, lse):
        w = torch.zeros(p.k_cache.shape[:3], device=cuda_device)
        out = fam.paged_prefix_attention(x.q, x.k_cache, x.v_cache, *x.prefix, *x.where, True, 0.1, max_q_len=1)
        fam.paged_attention_weights(p.q, lse, p.k_cache, *p.where, w, True, 0.1)
        k, v = p.k_cache.clone(), p.v_cache.clone()
        lens, kept = fam.paged_cache_evict(k, v, w.clone(), p.table, p.lens, 1000, 10, return_kept=True)
        return out, w, kept, k.view(torch.uint8), v.view(torch.uint8)

    want = [calls(*a) for a in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in work]
    for _ in range(5):
        got = []
        for s, a in zip(streams, work):
            with torch.cuda.stream(s):
                got.append(calls(*a))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(x, y))


@pytest.mark.parametrize("head_dim,fp8", [(128, False), (256, True), (64, False)])
def test_blocks_of_one_and_two_key_tiles_in_turn(head_dim, fp8, cuda_device):
    """Sequences of at most 128 tokens leave the second key tile out, one after the other."""
    lens = [(300, 5, 90, 128, 1, 129, 60, 700, 3, 17, 255, 2)[i % 12] for i in range(150)]
    b = ref.Batch([1] * 150, lens, heads_q=8, heads_kv=4, head_dim=head_dim, page=32, fp8=fp8, device=cuda_device, seed=1)
    lse = ref_w.logsumexps(b, True, 0.1)
    old = torch.rand(b.k_cache.shape[:3], device=cuda_device)
    want, tol = ref_w.weights(b, lse, old, True, 0.1)
    for longest in (1, None):
        for _ in range(5):
            w = old.clone()
            fam.paged_attention_weights(b.q, lse, b.k_cache, *b.where, w, True, 0.1, k_scale=b.k_scale, max_q_len=longest)
            assert ((w.double() - want).abs() <= tol).all()
    ops.check_device_status(cuda_device)


def test_registered_operators(cuda_device):
    x = pre.PrefixBatch([1, 9], [50, 77], [200], [10], head_dim=64, device=cuda_device, garbage=0.0)
    args = (x.q, x.k_cache, x.v_cache, *x.prefix, *x.where, True, 0.1)
    out, lse = OPS.paged_prefix_attention(*args)
    want = fam.paged_prefix_attention(x.q, x.k_cache, x.v_cache, *x.prefix, *x.where, True, 0.1, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(OPS.paged_prefix_attention, args, test_utils=utils)
    w = torch.zeros(x.k_cache.shape[:3], device=cuda_device)
    torch.library.opcheck(OPS.paged_attention_weights, (x.q, lse, x.k_cache, *x.where, w, True, 0.1), test_utils=utils)
    torch.library.opcheck(OPS.paged_cache_evict, (x.k_cache, x.v_cache, w, x.table, x.lens, 40, 4, None, None),
                          test_utils=utils)
    version = w._version, x.k_cache._version
    OPS.paged_attention_weights(x.q, lse, x.k_cache, *x.where, w, True, 0.1)
    OPS.paged_cache_evict(x.k_cache, x.v_cache, w, x.table, x.lens, 40, 4, None, None)
    assert w._version > version[0] and x.k_cache._version > version[1]


def test_rows_of_any_layout_and_refused_outputs(cuda_device):
    x = pre.PrefixBatch([1, 9], [50, 77], [200], [10], head_dim=64, device=cuda_device, garbage=0.0)
    more = (x.k_cache, x.v_cache, *x.prefix, *x.where, True, 0.1)
    want = fam.paged_prefix_attention(x.q, *more)
    wide = torch.empty(*x.q.shape[:2], 67, dtype=x.q.dtype, device=cuda_device)[..., 1:65].copy_(x.q)
    permuted = x.q.transpose(0, 1).contiguous().transpose(0, 1)
    for q in (wide, permuted):
        assert torch.equal(fam.paged_prefix_attention(q, *more), want)
    for kw in (dict(out=torch.empty_like(wide)[..., :32]), dict(out=torch.empty_like(x.q).float()),
               dict(lse=torch.empty(10, 4, device=cuda_device)[:, :3]), dict(out=wide)):
        with pytest.raises(ValueError):
            fam.paged_prefix_attention(x.q, *more, **kw)


def test_beyond_32_bit_offsets(cuda_device):
    """Pages whose elements lie past 2^32: prefix, weights and eviction find them."""
    pages, page, d = 16500, 1024, 256
    k = torch.zeros(pages, 1, page, d, dtype=ref.FP8, device=cuda_device)
    v = torch.zeros_like(k)
    ks, vs = (torch.ones(pages, 1, page, device=cuda_device) for _ in range(2))
    g = torch.Generator(device=cuda_device).manual_seed(1)
    far = [pages - 1 - i for i in range(6)]
    for x in (k, v):
        x[far] = torch.randn(6, 1, page, d, device=cuda_device, generator=g).to(ref.FP8)

    class View:
        pass
    x = View()
    x.k_cache, x.v_cache, x.k_scale, x.v_scale = k, v, ks, vs
    ints = lambda y: torch.tensor(y, dtype=torch.int32, device=cuda_device)  # noqa: E731
    x.table, x.offsets, x.lens = ints([far[:3], far[3:5] + [0]]), ints([0, 1, 4]), ints([2500, 1100])
    x.prefix_table, x.prefix_offsets, x.prefix_lens = ints([far[5:]]), ints([0, 4]), ints([1000])
    x.q = torch.randn(4, 2, d, device=cuda_device, generator=g).to(FP16)
    scales = dict(k_scale=ks, v_scale=vs)
    out, lse = fam.paged_prefix_attention(x.q, k, v, x.prefix_table, x.prefix_offsets, x.prefix_lens, x.table, x.offsets,
                                          x.lens, True, 0.0625, return_lse=True, **scales)
    want, want_lse, tol, tol_lse = pre.attention(x, True, 0.0625)
    assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= tol_lse).all()
    w = torch.zeros(pages, 1, page, device=cuda_device)
    wanted, tol = ref_w.weights(x, lse, w, True, 0.0625)
    fam.paged_attention_weights(x.q, lse, k, x.table, x.offsets, x.lens, w, True, 0.0625, k_scale=ks)
    assert ((w.double() - wanted).abs() <= tol).all()
    before = [y[far[:5]].clone() for y in (k, v, w)]
    lens, kept = fam.paged_cache_evict(k, v, w, x.table, x.lens, 1050, 100, return_kept=True, **scales)
    small = ints([[0, 1, 2], [3, 4, 4]])
    want_lens, want_kept, moved = ref_e.evict(before, before[2], small, x.lens, 1050, 100)
    assert torch.equal(lens.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
    for y, z in zip((k, v, w), moved):
        assert torch.equal(ref_e.bits(y[far[:5]].cpu()).view(z.shape), z)
    ops.check_device_status(cuda_device)


# ---------------------------------------------------------------------------------- bounded waits
def _child_main(kind: str, head_dim: int, fp8: bool) -> None:
    """Calls of a library whose waits give up at once come back and say so; the product's go on working."""
    from flash_attn_npu_b200 import _native

    def use(lib):
        binding = paged._native_binding()
        binding.setup_more(*(ctypes.cast(getattr(lib, "fa_paged_" + name), ctypes.c_void_p).value for name in (
            "prefix_sm100", "prefix_workspace_bytes", "weights_sm100", "weights_workspace_bytes", "evict_sm100",
            "evict_workspace_bytes")))

    dev = torch.device("cuda", 0)
    word = ops.device_status_word(dev)
    product, short = _native.load(), ctypes.CDLL(str(build.variant_path("shortwait")))
    if kind.startswith("prefix"):
        n = 40 if kind == "prefix-two" else 3
        x = pre.PrefixBatch([1] * n, [300] * n, [5000], [n], heads_q=8, heads_kv=2, head_dim=head_dim, page=64, fp8=fp8,
                            device=dev)

        def call():
            return fam.paged_prefix_attention(x.q, x.k_cache, x.v_cache, *x.prefix, *x.where, True, 0.1, max_q_len=1,
                                              **x.scales)
        want, _, tol, _ = pre.attention(x, True, 0.1)
    elif kind == "evict":
        x = ref.Batch([0], [60000], heads_q=2, heads_kv=2, head_dim=head_dim, page=64, fp8=fp8, device=dev)
        w = torch.rand(x.k_cache.shape[:3], device=dev)

        def call():
            k, v = x.k_cache.clone(), x.v_cache.clone()
            scales = {n: None if y is None else y.clone() for n, y in x.scales.items()}
            fam.paged_cache_evict(k, v, w.clone(), x.table, x.lens, 30000, 10, **scales)
            return v.view(torch.uint8)
        held = [x.k_cache, x.v_cache]
        want = ref_e.evict(held, w, x.table, x.lens, 30000, 10)[2][1].to(dev).view(call().shape)
        tol = torch.zeros_like(want)
    else:
        counts, lens = ([1] * 40, [3000] * 40) if kind == "weights-one" else ([700] * 3, [1500] * 3)
        x = ref.Batch(counts, lens, heads_q=8, heads_kv=2, head_dim=head_dim, page=64, fp8=fp8, device=dev)
        lse = ref_w.logsumexps(x, True, 0.1)
        old = torch.zeros(x.k_cache.shape[:3], device=dev)

        def call():
            w = old.clone()
            fam.paged_attention_weights(x.q, lse, x.k_cache, *x.where, w, True, 0.1, k_scale=x.k_scale,
                                        max_q_len=max(counts))
            return w
        want, tol = ref_w.weights(x, lse, old, True, 0.1)
    use(short)
    code = 0
    for _ in range(100):  # (in a small call every wait may find what it waits for there already)
        call()
        torch.cuda.synchronize(dev)
        code = int(word.item())
        if code:
            break
    word.zero_()
    use(product)
    got = call()
    ops.check_device_status(dev)
    print("RESULT " + json.dumps({"status": code, "good": bool(((got.double() - want).abs() <= tol).all())}), flush=True)


@pytest.mark.parametrize("head_dim,fp8", [(128, False), (128, True), (256, True)])
@pytest.mark.parametrize("kind", ["prefix-two", "prefix-one", "weights-one", "weights-many", "evict"])
def test_wait_that_gives_up_is_reported(kind, head_dim, fp8, native_lib, cuda_device):
    from flash_attn_npu_b200 import _native
    build.build(variant="shortwait")  # no-op when up to date
    res = subprocess.run([sys.executable, __file__, "child", kind, str(head_dim), str(int(fp8))], cwd=str(REPO),
                         env=dict(os.environ, PYTHONPATH=f"{REPO}:{REPO}/tests"), capture_output=True, text=True,
                         timeout=300)
    assert res.returncode == 0, res.stderr[-3000:]
    line = [ln for ln in res.stdout.splitlines() if ln.startswith("RESULT ")][-1]
    assert json.loads(line[len("RESULT "):]) == {"status": _native.FA_ERR_DEVICE_TIMEOUT, "good": True}


if __name__ == "__main__":
    if len(sys.argv) > 1 and sys.argv[1] == "child":
        sys.path[:0] = [str(REPO), str(REPO / "tests")]
        _child_main(sys.argv[2], int(sys.argv[3]), sys.argv[4] == "1")
