// C-ABI front end of the attention weights (declared in include/fa_paged_sm100.h): checks, tensor maps,
// workspace layout, launch.
#include <algorithm>
#include <cmath>

#include "fa_paged_host.h"
#include "fa_paged_launch.h"
#include "fa_paged_weights_launch.h"

namespace fa {

// fa_fwd_api.cu
int encode_cache_map(CUtensorMap* map, const void* ptr, int dtype, int64_t pages, int64_t heads, int64_t rows,
                     int64_t head_dim, const int64_t st[3], int box_cols, int box_rows, int swz_bytes);
int encode_query_map(CUtensorMap* map, const void* ptr, int dtype, int64_t total, int64_t heads, int64_t head_dim,
                     const int64_t st[2], int box_cols, int box_heads, int box_tokens, int swz_bytes);

namespace {

// The cache as the checks of the other calls take it: there are no values.
FaPagedCache keys_of(const FaPagedWeightsArgs* a) {
  FaPagedCache c = a->cache;
  c.v = c.k;
  c.v_scale = c.k_scale;
  for (int d = 0; d < 3; ++d) c.v_stride[d] = c.k_stride[d];
  for (int d = 0; d < 2; ++d) c.v_scale_stride[d] = c.k_scale_stride[d];
  return c;
}

int check_weights(const FaPagedWeightsArgs* a) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(FaPagedWeightsArgs))) return FA_ERR_INVALID_ARG;
  const int rc = check_layout(keys_of(a), a->dtype, a->total);
  if (rc != FA_OK) return rc;
  if (a->heads_q <= 0 || a->heads_q % a->cache.heads_kv || a->max_q_len < 0 || a->heads_q > 32768)
    return FA_ERR_INVALID_ARG;
  if (a->total * a->heads_q > INT32_MAX / 2) return FA_ERR_INVALID_ARG;
  if (!std::isfinite(a->sm_scale)) return FA_ERR_INVALID_ARG;
  for (int d = 0; d < 2; ++d)
    if (a->weights_stride[d] <= 0 || a->weights_stride[d] % 4) return FA_ERR_MISALIGNED;
  return FA_OK;
}

int query_rows(int64_t head_dim, bool fp8) {
  if (head_dim <= 64) return WeightsGeo<64, false>::QN;
  if (head_dim == 128) return fp8 ? WeightsGeo<128, true>::QN : WeightsGeo<128, false>::QN;
  return fp8 ? WeightsGeo<256, true>::QN : WeightsGeo<256, false>::QN;
}

struct WeightsChoice {
  int grid;
  int64_t parts, bytes;  // workspace: notes, parts
};

WeightsChoice choose() {
  WeightsChoice c{};
  c.grid = sm_count_of_current();
  c.parts = up256(static_cast<int64_t>(sizeof(PagedWeightsNote)) * c.grid);
  c.bytes = up256(c.parts + 4 * 2 * kWeightsBlock * static_cast<int64_t>(c.grid));
  return c;
}

int weights(const FaPagedWeightsArgs* a, void* stream) {
  int rc = check_weights(a);
  if (rc != FA_OK) return rc;
  const FaPagedCache kv = keys_of(a);
  rc = check_cache(kv, a->dtype, a->total);
  if (rc != FA_OK) return rc;
  if (a->total == 0 || kv.seqs == 0) return FA_OK;
  if (!a->q || !a->lse || !a->weights || !a->workspace) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a->q) % 16 || reinterpret_cast<uintptr_t>(a->weights) % 16 ||
      reinterpret_cast<uintptr_t>(a->lse) % 4 || reinterpret_cast<uintptr_t>(a->workspace) % 256)
    return FA_ERR_MISALIGNED;
  if (a->q_stride[0] <= 0 || a->q_stride[1] <= 0 || a->q_stride[0] % 8 || a->q_stride[1] % 8)
    return FA_ERR_MISALIGNED;
  rc = check_device();
  if (rc != FA_OK) return rc;
  const WeightsChoice c = choose();
  if (a->workspace_bytes < c.bytes) return FA_ERR_INVALID_ARG;

  WeightsPlan plan{};
  plan.half = a->dtype == FA_DTYPE_FP16;
  plan.fp8 = kv.dtype == FA_DTYPE_FP8_E4M3;
  plan.grid = c.grid;
  plan.stream = static_cast<cudaStream_t>(stream);
  PagedWeightsParams& p = plan.params;
  p.seqs = seqs_of(kv, a->total, a->dev_status);
  p.row_lse = a->lse;
  p.weights = a->weights;
  p.k_scale = kv.k_scale;
  for (int d = 0; d < 2; ++d) {
    p.weights_stride[d] = a->weights_stride[d];
    p.k_scale_stride[d] = kv.k_scale_stride[d];
  }
  p.reset_new = a->reset_new ? 1 : 0;
  p.heads_kv = static_cast<int>(kv.heads_kv);
  p.group = static_cast<int>(a->heads_q / kv.heads_kv);
  p.group_inv = static_cast<uint32_t>((int64_t{1} << 32) / p.group + 1);
  p.head_dim = static_cast<int>(kv.head_dim);
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->sm_scale * kLog2e;
  // A query tile has as many whole tokens as fit, but no more than a sequence has (their rows are loaded
  // and multiplied); a larger group has its heads in several tiles.
  const int most = query_rows(kv.head_dim, plan.fp8);
  const int64_t longest = a->max_q_len ? std::min(a->max_q_len, a->total) : a->total;
  p.tile_heads = std::min(p.group, most);
  p.chunks = (p.group + most - 1) / most;
  p.tile_toks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most / p.tile_heads, longest)));
  // Items of one step are not cut, and there is nothing to join.
  p.whole_items = p.chunks == 1 && longest <= p.tile_toks;
  p.item_cost = p.whole_items ? 0 : 1;
  p.min_steps_log2 = p.whole_items ? 0 : 1;
  char* ws = static_cast<char*>(a->workspace);
  p.notes = reinterpret_cast<PagedWeightsNote*>(ws);
  p.parts = reinterpret_cast<float*>(ws + c.parts);

  const int d = static_cast<int>(kv.head_dim), swz = std::min(2 * d, 128);
  const int box = static_cast<int>(std::min<int64_t>(kv.page_size, 128));
  rc = encode_cache_map(&plan.tmK, kv.k, kv.dtype, kv.num_pages, kv.heads_kv, kv.page_size, kv.head_dim, kv.k_stride,
                        plan.fp8 ? d : swz / 2, box, plan.fp8 ? 16 : swz);
  if (rc == FA_OK)
    rc = encode_query_map(&plan.tmQ, a->q, a->dtype, a->total, a->heads_q, kv.head_dim, a->q_stride, std::min(d, 64),
                          p.tile_heads, p.tile_toks, swz);
  if (rc != FA_OK) return rc;
  switch (d) {
    case 16: return launch_weights_d16(plan);
    case 32: return launch_weights_d32(plan);
    case 64: return launch_weights_d64(plan);
    case 128: return launch_weights_d128(plan);
    default: return launch_weights_d256(plan);
  }
}

}  // namespace
}  // namespace fa

extern "C" {

int64_t fa_paged_weights_workspace_bytes(const FaPagedWeightsArgs* a) {
  const int rc = fa::check_weights(a);
  return rc != FA_OK ? rc : fa::choose().bytes;
}

int fa_paged_weights_sm100(const FaPagedWeightsArgs* a, void* stream) { return fa::weights(a, stream); }

}  // extern "C"
