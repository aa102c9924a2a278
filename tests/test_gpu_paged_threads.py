"""The C ABI of the paged calls from several threads at once, the first calls of the process among them.

A child process starts the threads together; each has a stream, a workspace and a batch of its own, and takes the
kernels in another order (ctypes lets go of the interpreter's lock meanwhile).  What is shared are the library's
records of which kernels and devices it has looked at.
"""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys
import threading

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu
THREADS, TURNS = 8, 6
KINDS = [(1, False), (8, False), (60, False), (1, True), (8, True), (60, True)]  # tokens a sequence, float8


def _args(b, heads_q):
    """Attention, with its outputs and workspace, and write of a batch's rows."""
    from flash_attn_npu_b200 import _native, paged
    a, w = _native.FaPagedAttnArgs(), _native.FaPagedCopyArgs()
    for x in (a, w):
        x.struct_size = ctypes.sizeof(type(x))
        c = x.cache
        c.k, c.v = b.k_cache.data_ptr(), b.v_cache.data_ptr()
        c.page_table, c.offsets, c.kv_lens = (t.data_ptr() for t in b.where)
        c.k_stride[:], c.v_stride[:] = b.k_cache.stride()[:3], b.v_cache.stride()[:3]
        if b.fp8:
            c.k_scale, c.v_scale = b.k_scale.data_ptr(), b.v_scale.data_ptr()
            c.k_scale_stride[:], c.v_scale_stride[:] = b.k_scale.stride()[:2], b.v_scale.stride()[:2]
        c.num_pages, c.heads_kv, c.page_size, c.head_dim = b.k_cache.shape
        c.seqs, c.table_cols = b.table.shape
        c.table_stride = b.table.stride(0)
        c.dtype = paged._CACHE_CODES[b.k_cache.dtype]
        x.total, x.dtype = b.total, paged._ROW_CODES[b.q.dtype]
    out, lse = torch.zeros_like(b.q), torch.zeros(b.q.shape[:2], device=b.q.device)
    a.q, a.o, a.lse = b.q.data_ptr(), out.data_ptr(), lse.data_ptr()
    a.q_stride[:], a.o_stride[:] = b.q.stride()[:2], out.stride()[:2]
    a.heads_q, a.causal, a.sm_scale = heads_q, 1, 0.1
    a.max_q_len = int(b.offsets.diff().max())
    w.k, w.v = (x.data_ptr() for x in b.rows)
    w.k_stride[:], w.v_stride[:] = (x.stride()[:2] for x in b.rows)
    return a, w, out, lse


def _child_main() -> None:
    import paged_ref as ref
    from flash_attn_npu_b200 import _native
    dev = torch.device("cuda", 0)
    lib = _native.load()
    work = []
    for t in range(THREADS):
        mine = []
        for i in range(len(KINDS)):
            count, fp8 = KINDS[(i + t) % len(KINDS)]
            b = ref.Batch([count] * 2, [300 + t, 1200], heads_q=8, heads_kv=2, head_dim=64, fp8=fp8, device=dev, seed=t)
            mine.append((b, *_args(b, 8), torch.empty(64 << 20, dtype=torch.uint8, device=dev)))
        work.append((mine, torch.cuda.Stream(dev)))
    torch.cuda.synchronize(dev)
    together = threading.Barrier(THREADS)
    codes = []

    def run(mine, stream):
        together.wait()
        for _ in range(TURNS):
            for _, a, w, _, _, space in mine:
                codes.append(lib.fa_paged_write_sm100(ctypes.byref(w), stream.cuda_stream))
                a.workspace, a.workspace_bytes = space.data_ptr(), space.numel()
                assert 0 < lib.fa_paged_workspace_bytes(ctypes.byref(a)) <= space.numel()
                codes.append(lib.fa_paged_attn_sm100(ctypes.byref(a), stream.cuda_stream))

    threads = [threading.Thread(target=run, args=x) for x in work]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    torch.cuda.synchronize(dev)
    assert len(codes) == 2 * THREADS * TURNS * len(KINDS) and not any(codes), codes
    for mine, _ in work:
        for b, a, _, out, lse, _ in mine:
            want, want_lse, tol, tol_lse = ref.attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales,
                                                         max_q_len=a.max_q_len)
            assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= tol_lse).all()


def test_threads_make_their_first_calls_together(native_lib, cuda_device):
    res = subprocess.run([sys.executable, __file__, "child"], cwd=str(REPO), env=dict(os.environ), capture_output=True,
                         text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-3000:]


if __name__ == "__main__":
    if len(sys.argv) > 1 and sys.argv[1] == "child":
        sys.path[:0] = [str(REPO), str(REPO / "tests")]
        _child_main()
