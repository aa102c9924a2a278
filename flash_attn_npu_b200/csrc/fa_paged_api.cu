// C-ABI front end of the paged attention (declared in include/fa_paged_sm100.h): checks, kernel
// choice, tensor maps, workspace layout, launch.
#include <algorithm>
#include <cmath>

#include "fa_paged_host.h"
#include "fa_paged_launch.h"
#include "fa_paged_rows.cuh"
#include "fa_paged_tile.cuh"

namespace fa {

// fa_fwd_api.cu: 4-D tiled map over [pages, heads, rows, head_dim].
int encode_cache_map(CUtensorMap* map, const void* ptr, int dtype, int64_t pages, int64_t heads,
                     int64_t rows, int64_t head_dim, const int64_t st[3], int box_cols,
                     int box_rows, int swz_bytes);
// fa_fwd_api.cu: 3-D tiled map over packed queries [total, heads, head_dim].
int encode_query_map(CUtensorMap* map, const void* ptr, int dtype, int64_t total, int64_t heads,
                     int64_t head_dim, const int64_t st[2], int box_cols, int box_heads,
                     int box_tokens, int swz_bytes);

namespace {

template <int D, bool FP8, int ROWS>
constexpr PagedInfo rows_info() {
  using G = RowsGeo<D, FP8, ROWS>;
  return PagedInfo{ROWS, G::KEYS, G::SPAN, FP8 ? G::SPAN : G::SPAN / 2};
}

// rows: of a block of the row kernel; 0: the tile kernel.
template <int D>
PagedInfo info_of(bool fp8, int rows) {
  if (rows == 0) {
    using G = TileGeo<D, false>;  // float8 tiles land as they are, without a swizzle
    return fp8 ? PagedInfo{128 * G::TILES, G::KEYS, 16, D}
               : PagedInfo{128 * G::TILES, G::KEYS, G::SWZ, G::SWZ / 2};
  }
  if (rows == 8) return fp8 ? rows_info<D, true, 8>() : rows_info<D, false, 8>();
  if constexpr (D <= 128) {
    if (rows == 32) return fp8 ? rows_info<D, true, 32>() : rows_info<D, false, 32>();
  }
  return fp8 ? rows_info<D, true, 16>() : rows_info<D, false, 16>();
}

PagedInfo info_for(int64_t head_dim, bool fp8, int rows) {
  switch (head_dim) {
    case 16: return info_of<16>(fp8, rows);
    case 32: return info_of<32>(fp8, rows);
    case 64: return info_of<64>(fp8, rows);
    case 128: return info_of<128>(fp8, rows);
    default: return info_of<256>(fp8, rows);
  }
}

int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

// What a call runs with, from its arguments alone.
struct Choice {
  int rows;  // of a block of the row kernel; 0: the tile kernel
  PagedInfo info;
  int grid;
  int64_t parts, lse, o, bytes;  // workspace offsets
};

int check_attn(const FaPagedAttnArgs* a) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(FaPagedAttnArgs)))
    return FA_ERR_INVALID_ARG;
  const int rc = check_layout(a->cache, a->dtype, a->total);
  if (rc != FA_OK) return rc;
  if (a->heads_q <= 0 || a->heads_q % a->cache.heads_kv || a->max_q_len < 0)
    return FA_ERR_INVALID_ARG;
  if (a->heads_q > 32768) return FA_ERR_INVALID_ARG;
  // rows of a sequence (tokens x query heads) are counted in 32 bits
  if (a->total * a->heads_q > INT32_MAX / 2) return FA_ERR_INVALID_ARG;
  if (!std::isfinite(a->sm_scale)) return FA_ERR_INVALID_ARG;
  return FA_OK;
}

Choice choose(const FaPagedAttnArgs* a) {
  Choice c{};
  const int64_t group = a->heads_q / a->cache.heads_kv;
  const int64_t longest = a->max_q_len ? std::min(a->max_q_len, a->total) : a->total;
  // Up to 32 rows a kv head every sequence is one block of the row kernel, which reads the cache
  // once; above that the tile kernel does so for 128 or 256 rows.  It needs a positive scale, and
  // a group that fits a tile.  At 32 rows (8 kv heads) the row kernel takes 44 us and the tile kernel
  // 59 for 16 sequences of 4096 tokens at head_dim 64, 65 and 66 at 128, 63 and 88 at 128 from float8,
  // 10.7 and 11.6 for one of 512; only 40 of 2048 in 16 bits go the other way (85 and 77).
  // At head_dim 256 that does not hold: blocks have 16 rows, so 17 to 32 rows are two of them, which
  // read the cache one after the other.  There 16 sequences of 4096 tokens take 216 us and 110 (float8: 239
  // and 129), 40 of 2048 270 and 137, one of 512 17 and 17.
  const int64_t most = longest * group;
  if (most > 32 && group <= 128 && a->sm_scale > 0.f) c.rows = 0;
  else if (most <= 8) c.rows = 8;
  else c.rows = most <= 16 || a->cache.head_dim > 128 ? 16 : 32;
  c.info = info_for(a->cache.head_dim, a->cache.dtype == FA_DTYPE_FP8_E4M3, c.rows);
  c.grid = sm_count_of_current();
  const int64_t rows = 2 * static_cast<int64_t>(c.info.rows) * c.grid;
  c.parts = 0;
  c.lse = up256(c.parts + static_cast<int64_t>(sizeof(PagedPart)) * c.grid);
  c.o = up256(c.lse + 4 * rows);
  c.bytes = up256(c.o + 4 * rows * a->cache.head_dim);
  return c;
}

}  // namespace

}  // namespace fa

extern "C" {

int64_t fa_paged_workspace_bytes(const FaPagedAttnArgs* a) {
  const int rc = fa::check_attn(a);
  return rc != FA_OK ? rc : fa::choose(a).bytes;
}

int fa_paged_attn_sm100(const FaPagedAttnArgs* a, void* stream) {
  int rc = fa::check_attn(a);
  if (rc == FA_OK) rc = fa::check_cache(a->cache, a->dtype, a->total);
  if (rc != FA_OK) return rc;
  if (a->total == 0 || a->cache.seqs == 0) return FA_OK;
  if (!a->q || !a->o || !a->lse || !a->workspace) return FA_ERR_INVALID_ARG;
  for (const void* x : {a->q, static_cast<const void*>(a->o)})
    if (reinterpret_cast<uintptr_t>(x) % 16) return FA_ERR_MISALIGNED;
  for (const int64_t* st : {a->q_stride, a->o_stride})
    if (st[0] <= 0 || st[1] <= 0 || st[0] % 8 || st[1] % 8) return FA_ERR_MISALIGNED;
  if (reinterpret_cast<uintptr_t>(a->lse) % 4 ||
      reinterpret_cast<uintptr_t>(a->workspace) % 256)
    return FA_ERR_MISALIGNED;
  rc = fa::check_device();
  if (rc != FA_OK) return rc;
  const fa::Choice c = fa::choose(a);
  if (a->workspace_bytes < c.bytes) return FA_ERR_INVALID_ARG;

  const FaPagedCache& kv = a->cache;
  fa::PagedPlan plan{};
  plan.half = a->dtype == FA_DTYPE_FP16;
  plan.fp8 = kv.dtype == FA_DTYPE_FP8_E4M3;
  plan.rows = c.rows;
  plan.grid = c.grid;
  plan.stream = static_cast<cudaStream_t>(stream);
  const fa::PagedInfo& info = c.info;
  const int box = static_cast<int>(std::min<int64_t>(kv.page_size, info.keys));
  rc = fa::encode_cache_map(&plan.tmK, kv.k, kv.dtype, kv.num_pages, kv.heads_kv, kv.page_size,
                            kv.head_dim, kv.k_stride, info.cols, box, info.span);
  if (rc == FA_OK)
    rc = fa::encode_cache_map(&plan.tmV, kv.v, kv.dtype, kv.num_pages, kv.heads_kv, kv.page_size,
                              kv.head_dim, kv.v_stride, info.cols, box, info.span);
  if (rc != FA_OK) return rc;

  fa::PagedAttnParams& p = plan.params;
  p.seqs = fa::seqs_of(kv, a->total, a->dev_status);
  p.q = a->q;
  p.o = a->o;
  p.lse = a->lse;
  for (int d = 0; d < 2; ++d) {
    p.q_stride[d] = a->q_stride[d];
    p.o_stride[d] = a->o_stride[d];
    p.k_scale_stride[d] = kv.k_scale_stride[d];
    p.v_scale_stride[d] = kv.v_scale_stride[d];
  }
  p.k_scale = kv.k_scale;
  p.v_scale = kv.v_scale;
  p.heads_kv = static_cast<int>(kv.heads_kv);
  p.group = static_cast<int>(a->heads_q / kv.heads_kv);
  p.group_inv = static_cast<uint32_t>((int64_t{1} << 32) / p.group + 1);
  p.head_dim = static_cast<int>(kv.head_dim);
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->sm_scale * fa::kLog2e;
  const bool tile = c.rows == 0;
  // Sequences of at most kWholeTiles tiles are not cut: the joining launch costs more (3 .. 10 us)
  // than the tiles that a CTA then takes one after the other (~0.5 us each in the row kernel,
  // ~1.3 us in the tile kernel), however many SMs have nothing to do.  (What is known here is the table's
  // width, so the same lengths behind a wider table are cut.)  Not cut, and cut, at head_dim 128: one token of
  // one sequence of 777 with 16 kv heads 8.3 and 10.2 us, with 8 kv heads 8.4 and 9.8; of 8 such sequences 9.1
  // and 12.1, of 64 40.6 and 43.4; 100 tokens of 4 sequences of 900 25 and 35, of 16 50 and 77 (float8: 64 and
  // 94); a prompt of 500 17 and 26.
  constexpr int64_t kWholeTiles = 8;
  p.whole_items = kv.table_cols * kv.page_size <= kWholeTiles * info.keys;
  p.min_steps_log2 = p.whole_items ? 0 : tile ? 2 : 1;
  // What an item costs besides its tiles, in tiles: at head_dim 128 with blocks of 32 rows 6500 cycles
  // where a tile takes 2000 to 2800, with 16 rows 5000 (other head dims go by the same counts, unmeasured).
  // Counted as one for all of them, drafts of 16 sequences
  // took 61.9 us instead of 56.7, single tokens of 64 and 40 sequences the same time.  In the tile
  // kernel 2 took 102 to 104 us and 3 took 105 to 108 for the mixed batch of fa_paged_tile.cuh; other
  // chunks differ by 2 % either way.
  p.item_cost = tile ? 2 : c.rows == 32 ? 4 : c.rows == 16 ? 2 : 1;
  p.pair_from = plan.fp8 ? 6 : 3;
  p.tile_toks = tile ? 128 / p.group : 0;
  p.tile_live = tile ? p.tile_toks * p.group : info.rows;
  char* ws = static_cast<char*>(a->workspace);
  p.parts = reinterpret_cast<fa::PagedPart*>(ws + c.parts);
  p.part_lse = reinterpret_cast<float*>(ws + c.lse);
  p.part_o = reinterpret_cast<float*>(ws + c.o);

  if (tile) {
    rc = fa::encode_query_map(&plan.tmQ, a->q, a->dtype, a->total, a->heads_q, kv.head_dim,
                              a->q_stride, static_cast<int>(std::min<int64_t>(kv.head_dim, 64)),
                              p.group, p.tile_toks, static_cast<int>(std::min<int64_t>(2 * kv.head_dim, 128)));
    if (rc != FA_OK) return rc;
    switch (kv.head_dim) {
      case 16: return fa::launch_tile_d16(plan);
      case 32: return fa::launch_tile_d32(plan);
      case 64: return fa::launch_tile_d64(plan);
      case 128: return fa::launch_tile_d128(plan);
      default: return fa::launch_tile_d256(plan);
    }
  }
  switch (kv.head_dim) {
    case 16: return fa::launch_rows_d16(plan);
    case 32: return fa::launch_rows_d32(plan);
    case 64: return fa::launch_rows_d64(plan);
    case 128: return fa::launch_rows_d128(plan);
    default: return fa::launch_rows_d256(plan);
  }
}

}  // extern "C"
