// Host-side checks shared by the entry points of the paged key/value cache.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "../../include/fa_paged_sm100.h"
#include "fa_paged_common.cuh"

namespace fa {

// FA_OK if the current device is an sm_100 part (fa_fwd_api.cu).
int check_device();
// Streaming multiprocessors of the current device (fa_fwd_api.cu).
int sm_count_of_current();

inline int log2_of(int64_t x) {
  int n = 0;
  while ((int64_t{1} << n) < x) ++n;
  return n;
}

// Sizes, types and strides of a cache against the packed rows' type.
inline int check_layout(const FaPagedCache& c, int dtype, int64_t total) {
  constexpr int64_t kMost = int64_t{1} << 30;
  if (dtype != FA_DTYPE_FP16 && dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED_DTYPE;
  if (c.dtype != dtype && c.dtype != FA_DTYPE_FP8_E4M3) return FA_ERR_UNSUPPORTED_DTYPE;
  if (c.head_dim != 16 && c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128 &&
      c.head_dim != 256)
    return FA_ERR_UNSUPPORTED_HEAD_DIM;
  if (c.page_size < 8 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)))
    return FA_ERR_INVALID_ARG;
  if (total < 0 || total > kMost || c.seqs < 0 || c.seqs > kMost || c.num_pages <= 0 ||
      c.num_pages > kMost || c.heads_kv <= 0 || c.heads_kv > 65536 || c.table_cols < 0)
    return FA_ERR_INVALID_ARG;
  if (c.table_cols * c.page_size > kMost) return FA_ERR_INVALID_ARG;  // positions are 32-bit
  const bool f8 = c.dtype == FA_DTYPE_FP8_E4M3;
  const int64_t unit = f8 ? 16 : 8;  // elements in 16 bytes
  for (const int64_t* st : {c.k_stride, c.v_stride})
    for (int d = 0; d < 3; ++d)
      if (st[d] <= 0 || st[d] % unit || st[d] >= (int64_t{1} << 38)) return FA_ERR_MISALIGNED;
  if (f8)
    for (const int64_t* st : {c.k_scale_stride, c.v_scale_stride})
      for (int d = 0; d < 2; ++d)
        if (st[d] <= 0 || st[d] % 4) return FA_ERR_MISALIGNED;
  return FA_OK;
}

// ... and its addresses.
inline int check_cache(const FaPagedCache& c, int dtype, int64_t total) {
  const int rc = check_layout(c, dtype, total);
  if (rc != FA_OK) return rc;
  if (!c.k || !c.v || !c.offsets || (c.seqs > 0 && !c.kv_lens) ||
      (c.seqs > 0 && c.table_cols > 0 && !c.page_table))
    return FA_ERR_INVALID_ARG;
  if (c.dtype == FA_DTYPE_FP8_E4M3 && (!c.k_scale || !c.v_scale)) return FA_ERR_INVALID_ARG;
  for (const void* x : {static_cast<const void*>(c.k), static_cast<const void*>(c.v),
                        static_cast<const void*>(c.k_scale), static_cast<const void*>(c.v_scale)})
    if (reinterpret_cast<uintptr_t>(x) % 16) return FA_ERR_MISALIGNED;
  return FA_OK;
}

inline PagedSeqs seqs_of(const FaPagedCache& c, int64_t total, int* status) {
  PagedSeqs s{};
  s.page_table = c.page_table;
  s.offsets = c.offsets;
  s.kv_lens = c.kv_lens;
  s.table_stride = c.table_stride;
  s.table_cols = static_cast<int>(c.table_cols);
  s.seqs = static_cast<int>(c.seqs);
  s.num_pages = static_cast<int>(c.num_pages);
  s.page_log2 = log2_of(c.page_size);
  s.total = static_cast<int>(total);
  s.status = status;
  return s;
}

}  // namespace fa
