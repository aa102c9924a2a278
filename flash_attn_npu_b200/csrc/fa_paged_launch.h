// Launch plan of a paged attention call, shared by the C-ABI front end (fa_paged_api.cu) and the
// translation units that hold the kernel instantiations (fa_paged_rows_d*.cu).
#pragma once

#include <atomic>

#include "../../include/fa_paged_sm100.h"
#include "fa_paged_attn.cuh"

namespace fa {

// Facts of a kernel that the host needs: rows of a block, keys of a tile, and the boxes of its
// TMA copies.
struct PagedInfo {
  int rows, keys;
  int span;  // bytes of a copied row: the swizzle width
  int cols;  // elements of a copied row
};

struct PagedPlan {
  CUtensorMap tmQ, tmK, tmV;  // tmQ: tile kernel
  PagedLevelParams params;  // (its own part: calls behind shared prefixes)
  bool half;  // q and the output are fp16 (else bf16)
  bool fp8;
  int rows;   // row kernel: rows of a block (8, 16 or 32)
  int grid;
  cudaStream_t stream;
};

// What a call runs with, from its arguments alone.
struct PagedChoice {
  int rows;  // of a block of the row kernel; 0: the tile kernel
  PagedInfo info;
  int grid;
  int64_t parts, lse, o, bytes;  // workspace offsets
};

inline int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

// fa_paged_api.cu: sizes and types; pointers; the kernel for a call, or for that many rows a kv head of a
// sequence; whether the tile kernel can take it; the launch that it takes (the workspace at `ws`); and that
// launch.
int check_attn(const FaPagedAttnArgs* a);
int check_attn_pointers(const FaPagedAttnArgs* a);
PagedChoice choose_attn(const FaPagedAttnArgs* a);
PagedChoice choose_for_rows(const FaPagedAttnArgs* a, int64_t most);
bool tile_kernel_takes(const FaPagedAttnArgs* a);
int plan_attn(const FaPagedAttnArgs* a, const PagedChoice& c, char* ws, cudaStream_t stream, PagedPlan& plan);
int launch_attn(const PagedPlan& plan);

int launch_tile_d16(const PagedPlan& plan);
int launch_tile_d32(const PagedPlan& plan);
int launch_tile_d64(const PagedPlan& plan);
int launch_tile_d128(const PagedPlan& plan);
int launch_tile_d256(const PagedPlan& plan);
int launch_rows_d16(const PagedPlan& plan);
int launch_rows_d32(const PagedPlan& plan);
int launch_rows_d64(const PagedPlan& plan);
int launch_rows_d128(const PagedPlan& plan);
int launch_rows_d256(const PagedPlan& plan);
int launch_levels_tile_d16(const PagedPlan& plan);
int launch_levels_tile_d32(const PagedPlan& plan);
int launch_levels_tile_d64(const PagedPlan& plan);
int launch_levels_tile_d128(const PagedPlan& plan);
int launch_levels_tile_d256(const PagedPlan& plan);
int launch_levels_rows_d16(const PagedPlan& plan);
int launch_levels_rows_d32(const PagedPlan& plan);
int launch_levels_rows_d64(const PagedPlan& plan);
int launch_levels_rows_d128(const PagedPlan& plan);
int launch_levels_rows_d256(const PagedPlan& plan);

// (Calls of several threads may meet in the two below: what they remember is atomic, and only successes
// are remembered.)

// A kernel's opt-in to more than 48 KB of shared memory, made once per device: the call costs as
// much as a small part of a launch.
struct SmemOptIn {
  std::atomic<bool> done[16] = {};
  bool operator()(const void* kernel, int bytes) {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
    if (dev >= 0 && dev < 16 && done[dev].load(std::memory_order_acquire)) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    if (dev >= 0 && dev < 16) done[dev].store(true, std::memory_order_release);
    return true;
  }
};

// Whether a kernel was built with `regs` registers a thread: setmaxnreg redistributes exactly the launch
// allocation, so a build that differs is refused.
struct RegsMatch {
  std::atomic<bool> known{false};
  bool operator()(const void* kernel, int regs) {
    if (known.load(std::memory_order_relaxed)) return true;
    cudaFuncAttributes attr{};
    if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    if (attr.numRegs != regs) return false;
    known.store(true, std::memory_order_relaxed);
    return true;
  }
};

// Launch with programmatic dependence on the kernel before it in the stream (see
// wait_for_launch_before): only launch latency and set-up overlap.
template <typename... Params, typename... Args>
int launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, int smem,
                     cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess) return 0;
  (void)cudaGetLastError();
  return -7;
}

}  // namespace fa
