"""`torch.ops.flash_attn_b200.paged_*`: fake implementations on the CPU, and on the GPU the same
results as the calls they wrap, the operator checks, and a captured step of all three."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import paged_ref as ref
from flash_attn_npu_b200 import paged, torch_op  # noqa: F401  (registers the operators)

OPS = torch.ops.flash_attn_b200
BF16, FP16 = torch.bfloat16, torch.float16


def _batch(**kw):
    return ref.Batch([1, 3, 0, 40], [20, 30, 8, 41], **kw)


def _attend(b, q=None):
    return (b.q if q is None else q, b.k_cache, b.v_cache, *b.where, True, 0.1, b.k_scale, b.v_scale)


def _write(b):
    return (*b.rows, b.k_cache, b.v_cache, *b.where, b.k_scale, b.v_scale)


def _read(b, dtype=None):
    return (b.k_cache, b.v_cache, *b.where, b.total, b.k_scale, b.v_scale, dtype)


# ----------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("fp8", [False, True])
def test_fake_shapes_on_meta(fp8):
    b = _batch(fp8=fp8, dtype=FP16, device="meta")
    b.total = b.q.shape[0]
    out, lse = OPS.paged_attention(*_attend(b))
    assert out.shape == b.q.shape and out.dtype == FP16 and out.stride() == b.q.stride()
    assert lse.shape == b.q.shape[:2] and lse.dtype == torch.float32 and lse.is_contiguous()
    assert OPS.paged_cache_write(*_write(b)) is None
    for dtype in (None, FP16):
        k, v = OPS.paged_cache_read(*_read(b, dtype))
        assert k.shape == v.shape == b.rows[0].shape and k.dtype == v.dtype
        assert k.dtype == (BF16 if fp8 and dtype is None else FP16)


def test_fake_layout_of_the_output():
    b = _batch(device="meta")
    n, h, d = b.q.shape
    q = torch.empty(h, n, d, dtype=BF16, device="meta").transpose(0, 1)
    assert OPS.paged_attention(*_attend(b, q))[0].stride() == q.stride()
    q = torch.empty(n, h, d + 1, dtype=BF16, device="meta")[..., :d]
    assert OPS.paged_attention(*_attend(b, q))[0].is_contiguous()


def test_fake_mode_and_refusals():
    with FakeTensorMode():
        k, v, ks, vs = paged.empty_cache(8, 16, 2, 64, ref.FP8, "cpu")
        table, offsets, lens = (torch.zeros(s, dtype=torch.int32) for s in ((3, 2), 4, 3))
        q = torch.empty(5, 4, 64, dtype=BF16)
        out, lse = OPS.paged_attention(q, k, v, table, offsets, lens, True, 0.1, ks, vs, 2)
        assert out.shape == q.shape and lse.shape == (5, 4)
    b = _batch(device="meta")
    with pytest.raises(ValueError, match="multiple of heads_kv"):
        OPS.paged_attention(*_attend(b, b.q[:, :3]))
    with pytest.raises(ValueError, match="no other"):
        OPS.paged_cache_write(*_write(b)[:-2], torch.empty(b.k_cache.shape[:3], device="meta"),
                              torch.empty(b.k_cache.shape[:3], device="meta"))


# ----------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_same_results_as_the_calls(fp8, cuda_device):
    b, c = (_batch(fp8=fp8, garbage=0.0, device=cuda_device) for _ in range(2))
    OPS.paged_cache_write(*_write(b))
    paged.write(*_write(c))
    for x, y in ((b.k_cache, c.k_cache), (b.v_cache, c.v_cache)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for x, y in zip(OPS.paged_attention(*_attend(b)), paged.attention(*_attend(c))):
        assert torch.equal(x, y)
    for x, y in zip(OPS.paged_cache_read(*_read(b)), paged.read(*_read(c))):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_opcheck_schema_and_fake(fp8, cuda_device):
    b = _batch(fp8=fp8, garbage=0.0, device=cuda_device)
    # (torch's schema check compares the arguments before and after with arithmetic that float8 lacks)
    tests = ("test_faketensor",) if fp8 else ("test_schema", "test_faketensor")
    for op, args in ((OPS.paged_attention, _attend(b)), (OPS.paged_cache_read, _read(b)),
                     (OPS.paged_cache_write, _write(b))):
        torch.library.opcheck(op, args, test_utils=tests)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_captured_step(fp8, cuda_device):
    """Write, attention and read recorded once, replayed on new rows in the captured buffers."""
    b = _batch(fp8=fp8, garbage=0.0, device=cuda_device)

    def step():
        OPS.paged_cache_write(*_write(b))
        return *OPS.paged_attention(*_attend(b)), *OPS.paged_cache_read(*_read(b))

    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream(cuda_device).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6):
        n = _batch(fp8=fp8, garbage=0.0, seed=seed)
        b.q.copy_(n.q)
        for x, y in zip(b.rows, n.rows):
            x.copy_(y)
        graph.replay()
        again = [x.clone() for x in got]
        want = step()
        for x, y in zip(again, want):
            assert torch.equal(x, y)
        k = ref.dequantise(*ref.quantise(b.rows[0])) if fp8 else b.rows[0].double()
        assert torch.equal(again[2].double(), k.to(BF16).double())
    del graph
