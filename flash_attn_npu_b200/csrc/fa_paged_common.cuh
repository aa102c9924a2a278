// What the kernels of the paged key/value cache share: the view of the cache and the sequences,
// the lookup of a token's place, and the division of an attention call's work among CTAs.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace fa {

constexpr int kStatusPageTable = -10;  // FA_ERR_PAGE_TABLE

// Sequences and their pages, as the kernels see them.
struct PagedSeqs {
  const int* page_table;
  const int* offsets;
  const int* kv_lens;
  int64_t table_stride;
  int table_cols;
  int seqs;
  int num_pages;
  int page_log2;
  int total;  // rows of the packed tensors
  int* status;
};

// A load of what an earlier kernel may have written.  Not through the read-only path: this kernel may
// have been brought up before that one ended (programmatic dependent launch), so the data may change
// within its lifetime.
template <typename T>
__device__ __forceinline__ T fresh(const T* p) {
  return *p;
}

__device__ __forceinline__ void report(int* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// Rows of sequence b in the packed tensors, kept inside [0, total].
__device__ __forceinline__ void seq_rows(const PagedSeqs& s, int b, int& first, int& count) {
  const int a = fresh(s.offsets + b), z = fresh(s.offsets + b + 1);
  first = min(max(a, 0), s.total);
  count = max(min(z, s.total) - first, 0);
}

// Length of sequence b in the cache, kept inside what its table row can name.
__device__ __forceinline__ int seq_len(const PagedSeqs& s, int b) {
  const int64_t cap = static_cast<int64_t>(s.table_cols) << s.page_log2;
  const int n = fresh(s.kv_lens + b);
  return n < 0 ? 0 : static_cast<int>(n < cap ? n : cap);
}

// Entry of the page table for a position inside sequence b, not looked at yet, and what it names: a
// page of the cache (0, and a report, where it is none).
__device__ __forceinline__ int page_entry(const PagedSeqs& s, int b, int pos) {
  return fresh(s.page_table + b * s.table_stride + (pos >> s.page_log2));
}
__device__ __forceinline__ int checked_page(const PagedSeqs& s, int entry) {
  if (static_cast<uint32_t>(entry) < static_cast<uint32_t>(s.num_pages)) return entry;
  report(s.status, kStatusPageTable);
  return 0;
}

// Page that holds position `pos` of sequence b, or -1 where there is none.
__device__ __forceinline__ int page_of(const PagedSeqs& s, int b, int pos) {
  const int col = pos >> s.page_log2;
  if (pos < 0 || col >= s.table_cols) return -1;
  const int page = page_entry(s, b, pos);
  return page >= 0 && page < s.num_pages ? page : -1;
}

template <typename T>
struct Cvt16;
template <>
struct Cvt16<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
};
template <>
struct Cvt16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
};

// Two float8 e4m3 values (low byte first) as two halves; exact, NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint16_t x) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(x));
  return d;
}

// round_e4m3 of two floats, `lo` in the low byte; NaN stays NaN, magnitudes are at most 448.
__device__ __forceinline__ uint32_t pack2_e4m3(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}

}  // namespace fa
