"""`torch.ops.flash_attn_b200`: the library's calls registered as PyTorch custom operators.

`fwd` wraps `ops.forward` (the C-ABI launch on the current stream) so the kernel can sit
inside code that PyTorch traces or captures: a fake implementation gives output shapes,
dtypes and strides without running anything (meta tensors, FakeTensorMode, torch.compile
graphs with the operator left opaque), and the launch itself is capture-safe (no allocation in
the C ABI, no host synchronisation), so it can be recorded into a CUDA graph.

    out, lse = torch.ops.flash_attn_b200.fwd(q, k, v, causal, sm_scale, 0, 0, 0, 0)

Arguments follow `ops.forward`: the last four are BLOCK_M, BLOCK_N, NUM_STAGES,
PERSISTENT_CTAS, each 0 for the library default.

`paged_attention`, `paged_cache_write` and `paged_cache_read` are the calls of `paged` in the same
way.  The write is registered as one that mutates the cache (and the scales of a float8 one), and
returns nothing; its scales have no default (a mutated argument must be there), None for a 16-bit
cache.

    out, lse = torch.ops.flash_attn_b200.paged_attention(q, k_cache, v_cache, page_table, offsets,
                                                         kv_lens, causal, sm_scale)
"""
from __future__ import annotations

import torch

from . import ops, paged


def _out_like(q: torch.Tensor) -> torch.Tensor:
    """Output allocation rule of `ops.forward` from shapes and strides alone: q's layout when a
    TMA tensor map can describe it (unit inner stride, 16-byte strides), else contiguous."""
    eb = q.element_size()
    ok = q.stride(-1) == 1 and all(
        q.shape[d] <= 1 or (q.stride(d) * eb) % 16 == 0 for d in range(q.ndim - 1))
    return torch.empty_like(q) if ok else q.new_empty(q.shape)


@torch.library.custom_op("flash_attn_b200::fwd", mutates_args=())
def fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool, sm_scale: float,
        block_m: int = 0, block_n: int = 0, num_stages: int = 0,
        persistent_ctas: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.forward(q, k, v, causal, sm_scale, block_m=block_m, block_n=block_n,
                       num_stages=num_stages, persistent_ctas=persistent_ctas)


@fwd.register_fake
def _fwd_fake(q, k, v, causal, sm_scale, block_m=0, block_n=0, num_stages=0,
              persistent_ctas=0):
    ops.validate_layout(q, k, v)
    z, h, n_ctx, _ = q.shape
    return _out_like(q), q.new_empty((z, h, n_ctx), dtype=torch.float32)


@torch.library.custom_op("flash_attn_b200::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    page_table: torch.Tensor, offsets: torch.Tensor, kv_lens: torch.Tensor,
                    causal: bool, sm_scale: float, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None,
                    max_q_len: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    return paged.attention(q, k_cache, v_cache, page_table, offsets, kv_lens, causal, sm_scale,
                           k_scale, v_scale, max_q_len)


@paged_attention.register_fake
def _paged_attention_fake(q, k_cache, v_cache, page_table, offsets, kv_lens, causal, sm_scale,
                          k_scale=None, v_scale=None, max_q_len=None):
    paged.validate_attention(q, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale,
                             max_q_len)
    return paged.empty_rows(q), q.new_empty(q.shape[:2], dtype=torch.float32)


@torch.library.custom_op("flash_attn_b200::paged_cache_write",
                         mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def paged_cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, page_table: torch.Tensor, offsets: torch.Tensor,
                      kv_lens: torch.Tensor, k_scale: torch.Tensor | None,
                      v_scale: torch.Tensor | None) -> None:
    paged.write(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)


@paged_cache_write.register_fake
def _paged_cache_write_fake(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale):
    paged.validate_copy(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)


@torch.library.custom_op("flash_attn_b200::paged_cache_read", mutates_args=())
def paged_cache_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                     offsets: torch.Tensor, kv_lens: torch.Tensor, total: int,
                     k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                     dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    return paged.read(k_cache, v_cache, page_table, offsets, kv_lens, total, k_scale, v_scale, dtype)


@paged_cache_read.register_fake
def _paged_cache_read_fake(k_cache, v_cache, page_table, offsets, kv_lens, total, k_scale=None,
                           v_scale=None, dtype=None):
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype == paged.FP8 else k_cache.dtype
    k = k_cache.new_empty((total, k_cache.shape[1], k_cache.shape[3]), dtype=dtype)
    v = torch.empty_like(k)
    paged.validate_copy(k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
    return k, v
