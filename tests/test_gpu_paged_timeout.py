"""The paged attention kernels' bounded waits, exercised without a fault, a hang or a missing barrier.

The test library `libfa_sm100_shortwait.so` is the product source built with a limit of zero for
waits on the pipeline (see test_gpu_timeout.py).  Some wait on a tile from global memory is certain to
give up.  All roles then fall through to the teardown, which drains copies and MMAs under the long limit.
A child process checks that the launches return, that the status word reads FA_ERR_DEVICE_TIMEOUT, and that
the context goes on working: the product library gives the oracle's results right behind.
"""
from __future__ import annotations

import ctypes
import json
import os
import subprocess
import sys

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu

# what runs: new tokens and lengths of the sequences
KINDS = {"rows": ([1] * 40, [3000] * 40),
         "rows-cut": ([1] * 3, [20000] * 3),
         "tile": ([700] * 12, [1500] * 12),
         "tile-pairs": ([20] * 8, [6000] * 8)}


def _child_main(kind: str, head_dim: int, fp8: bool) -> None:
    import paged_ref as ref
    from flash_attn_npu_b200 import _native, build, ops, paged

    def use(lib):
        binding = paged._native_binding()
        binding.setup(*(ctypes.cast(getattr(lib, "fa_paged_" + name), ctypes.c_void_p).value for name in (
            "attn_sm100", "workspace_bytes", "write_sm100", "read_sm100")))

    dev = torch.device("cuda", 0)
    counts, lens = KINDS[kind]
    b = ref.Batch(counts, lens, heads_q=8, heads_kv=2, head_dim=head_dim, page=64, fp8=fp8, device=dev)
    word = ops.device_status_word(dev)
    product, short = _native.load(), ctypes.CDLL(str(build.variant_path("shortwait")))
    use(short)
    paged.attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales, max_q_len=max(counts))
    torch.cuda.synchronize(dev)
    code = int(word.item())
    word.zero_()
    use(product)
    out, lse = paged.attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales, max_q_len=max(counts))
    want, want_lse, tol, tol_lse = ref.attention(b.q, b.k_cache, b.v_cache, *b.where, True, 0.1, **b.scales,
                                                 max_q_len=max(counts))
    ops.check_device_status(dev)
    good = bool(((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= tol_lse).all())
    print("RESULT " + json.dumps({"status": code, "good": good}), flush=True)


@pytest.mark.parametrize("head_dim,fp8", [(128, False), (128, True), (256, True)])
@pytest.mark.parametrize("kind", list(KINDS))
def test_wait_that_gives_up_is_reported(kind, head_dim, fp8, native_lib, cuda_device):
    from flash_attn_npu_b200 import _native, build
    build.build(variant="shortwait")  # no-op when up to date
    res = subprocess.run([sys.executable, __file__, "child", kind, str(head_dim), str(int(fp8))], cwd=str(REPO),
                         env=dict(os.environ), capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-3000:]
    line = [ln for ln in res.stdout.splitlines() if ln.startswith("RESULT ")][-1]
    assert json.loads(line[len("RESULT "):]) == {"status": _native.FA_ERR_DEVICE_TIMEOUT, "good": True}


if __name__ == "__main__":
    if len(sys.argv) > 1 and sys.argv[1] == "child":
        sys.path[:0] = [str(REPO), str(REPO / "tests")]
        _child_main(sys.argv[2], int(sys.argv[3]), sys.argv[4] == "1")
