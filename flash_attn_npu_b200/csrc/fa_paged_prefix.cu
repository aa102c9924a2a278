// Attention of a batch whose sequences share long prefixes (fa_paged_prefix_sm100 of
// include/fa_paged_sm100.h).  A row attends to the keys P of its group's prefix and to the keys S of its
// own sequence; with l_X = log2 sum_{j in X} 2^(s_j) and O_X the softmax average of the values over X,
//   l = log2(2^l_P + 2^l_S),   O = 2^(l_P - l) O_P + 2^(l_S - l) O_S ,
// which holds for any division of the keys, down to the parts that CTAs hold.
//
// A prefix is attended to by all rows of its group at once, as one sequence without a causal mask: its
// keys and values are read once for the group, and its products have rows enough for the tensor cores.
// So a call runs the paged attention kernels over the same packed rows twice, for the prefixes and for the
// sequences' own tokens (the levels), and joins a row's parts.  In decoding the first is work for the tile
// kernel, bound by its products, and the second for the row kernel, bound by memory: two launches that run
// side by side (programmatic dependent launch; `begin` in fa_paged_attn.cuh), each on its share of the SMs
// by what the levels weigh, which the kernels work out from the lengths, as these are device data.  Where
// one kernel suits both levels, one launch has the prefixes and the sequences in one line.
//
// Measured: 4 single tokens behind 1000 tokens (16 heads x 128) 12 us, launches and their loads; 64 behind 8191
// with 100 to 2000 of their own (32 / 8 heads x 128) 80 us, 4.1 TB/s; 40 drafts of 1 to 5 tokens behind three
// prefixes of up to 20,000 in float8 163 us, the row kernel's chain in 32-row blocks; 6 chunks of 200 to 700
// tokens behind 6001 (16 / 4 heads x 64) 127 us, 510 TFLOP/s, where exponentials take 56.
//
// The parts, their logsumexps and the join are fp32.  The probabilities meet the values in 16 bits, as in the
// kernels' ordinary calls, since that is what the tensor cores multiply: bf16 outputs are 2.3e-3 off (root mean
// square, relative) where one rounding of the exact result is 1.7e-3.
#include <algorithm>

#include "fa_paged_host.h"
#include "fa_paged_launch.h"

namespace fa {
namespace {

// A level's parts, as the kernel that held it left them.
struct JoinLevel {
  const float* part_o;
  const float* part_lse;
  const int* offsets;
  int seqs;
  int slot_rows;  // rows of a slot
  int ctas;
};

struct JoinParams {
  JoinLevel level[2];
  const float* whole_o;   // as in PagedLevelParams
  const float* whole_lse;
  const uint32_t* where;
  void* o;
  float* lse;
  int64_t o_stride[2];
  int rows;  // total * heads_q
  int heads_q;
};

constexpr int kJoinThreads = 128;

// D / 4 threads to a row, four columns each, times PS groups of them that take every PS-th part.
template <typename T, int D, int PS>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ JoinParams p) {
  constexpr int TPR = D / 4;
  constexpr int ROWS = kJoinThreads / (TPR * PS);
  __shared__ float4 s_o[PS > 1 ? kJoinThreads : 1];
  __shared__ float2 s_ml[PS > 1 ? PS * ROWS : 1];
  const int col = threadIdx.x % TPR, split = threadIdx.x / TPR % PS, r = threadIdx.x / (TPR * PS);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + r;
  let_next_launch();
  wait_for_launch_before();
  const int tok = static_cast<int>(min(row, static_cast<int64_t>(p.rows - 1)) / p.heads_q);
  int n[2], at[2];      // parts of each level, and the slot of the first
  uint32_t in_slot[2];
  bool live = row < p.rows;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const JoinLevel& v = p.level[x];
    const bool in = tok >= fresh(v.offsets) && tok < fresh(v.offsets + v.seqs);
    if (x == 1) live = live && in;
    const uint32_t w = in && live ? fresh(p.where + x * static_cast<int64_t>(p.rows) + row) : 0u;
    // (what a kernel that gave up has left may be any bits)
    const int first = min(static_cast<int>(w >> 10 & 1023), v.ctas - 1);
    n[x] = !in ? 0 : (w & 1023) == 0 ? 1 : min(static_cast<int>(w & 1023), v.ctas - first);
    at[x] = (w & 1023) == 0 ? -1 : first;
    in_slot[x] = min(w >> 20, static_cast<uint32_t>(v.slot_rows - 1));
  }
  const int count = live ? n[0] + n[1] : 0;
  // part i: its logsumexp, and its O
  auto part = [&](int i, const float*& o) -> float {
    const int x = i >= n[0];
    const JoinLevel& v = p.level[x];
    if (x) i -= n[0];
    if (at[x] < 0) {
      const int64_t y = x * static_cast<int64_t>(p.rows) + row;
      o = p.whole_o + y * D;
      return fresh(p.whole_lse + y);
    }
    const int64_t slot = i == 0 ? 2 * static_cast<int64_t>(at[x]) + 1 : 2 * static_cast<int64_t>(at[x] + i);
    const int64_t y = slot * v.slot_rows + in_slot[x];
    o = v.part_o + y * D;
    return fresh(v.part_lse + y);
  };
  // Four parts at a time, so that what they say and what they hold are on their way together; O is kept
  // relative to the largest logsumexp so far.
  constexpr int AT_ONCE = 4;
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = split; i < count; i += AT_ONCE * PS) {
    float l[AT_ONCE];
    float4 v[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const float* from = nullptr;
      l[u] = -INFINITY;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i + u * PS < count) {
        l[u] = part(i + u * PS, from);
        v[u] = fresh(reinterpret_cast<const float4*>(from) + col);
      }
    }
    float to = top;
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) to = fmaxf(to, l[u]);
    const float base = to == -INFINITY ? 0.f : to;
    const float f = top == -INFINITY ? 0.f : exp2f(top - base);
    sum *= f;
    acc.x *= f;
    acc.y *= f;
    acc.z *= f;
    acc.w *= f;
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const float w = exp2f(l[u] - base);
      if (w == 0.f) continue;  // a part without keys for the row may have left no values
      sum += w;
      acc.x += w * v[u].x;
      acc.y += w * v[u].y;
      acc.z += w * v[u].z;
      acc.w += w * v[u].w;
    }
    top = to;
  }
  if constexpr (PS > 1) {
    s_o[threadIdx.x] = acc;
    if (col == 0) s_ml[r * PS + split] = make_float2(top, sum);
    __syncthreads();
    if (split != 0) return;
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PS; ++i) top = fmaxf(top, s_ml[r * PS + i].x);
    sum = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const float2 ml = s_ml[r * PS + i];
      const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
      const float4 v = s_o[threadIdx.x + i * TPR];
      sum += w * ml.y;
      acc.x += w * v.x;
      acc.y += w * v.y;
      acc.z += w * v.z;
      acc.w += w * v.w;
    }
  }
  if (!live) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int head = static_cast<int>(row - static_cast<int64_t>(tok) * p.heads_q);
  T* out = static_cast<T*>(p.o) + tok * p.o_stride[0] + head * p.o_stride[1] + 4 * col;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2(acc.x * inv, acc.y * inv, static_cast<T*>(nullptr)),
                                              pack2(acc.z * inv, acc.w * inv, static_cast<T*>(nullptr)));
  if (col == 0) p.lse[row] = (top + log2f(sum)) * kLn2;  // (no key: -inf)
}

template <typename T, int D, int PS>
int launch_join(const JoinParams& p, cudaStream_t stream) {
  constexpr int ROWS = kJoinThreads / (D / 4 * PS);
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(p.rows) + ROWS - 1) / ROWS);
  return launch_dependent(paged_join_kernel<T, D, PS>, dim3(blocks), kJoinThreads, 0, stream, p);
}

template <typename T>
int join(const JoinParams& p, int64_t head_dim, bool split, cudaStream_t stream) {
  switch (head_dim) {
    case 16: return split ? launch_join<T, 16, 4>(p, stream) : launch_join<T, 16, 1>(p, stream);
    case 32: return split ? launch_join<T, 32, 4>(p, stream) : launch_join<T, 32, 1>(p, stream);
    case 64: return split ? launch_join<T, 64, 4>(p, stream) : launch_join<T, 64, 1>(p, stream);
    case 128: return split ? launch_join<T, 128, 4>(p, stream) : launch_join<T, 128, 1>(p, stream);
    default: return split ? launch_join<T, 256, 2>(p, stream) : launch_join<T, 256, 1>(p, stream);
  }
}

// The prefixes as the sequences of a call of their own.
FaPagedAttnArgs of_prefixes(const FaPagedPrefixArgs* a) {
  FaPagedAttnArgs x = a->attn;
  x.cache.page_table = a->prefix_table;
  x.cache.offsets = a->prefix_offsets;
  x.cache.kv_lens = a->prefix_lens;
  x.cache.table_stride = a->prefix_stride;
  x.cache.table_cols = a->prefix_cols;
  x.cache.seqs = a->prefixes;
  x.max_q_len = a->max_prefix_q_len;
  x.causal = 0;
  return x;
}

int check_prefix(const FaPagedPrefixArgs* a) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(FaPagedPrefixArgs))) return FA_ERR_INVALID_ARG;
  const int rc = check_attn(&a->attn);
  if (rc != FA_OK) return rc;
  const FaPagedAttnArgs x = of_prefixes(a);
  return check_attn(&x);
}

// One kernel for both levels, where both have few rows or the own tokens have many, else the tile kernel
// for the prefixes beside the row kernel for the own tokens.
struct PrefixChoice {
  int launches;
  bool lone_tile;  // the rows of a prefix fit one query tile
  PagedChoice kernel[2];
  int64_t own[2], whole_o, whole_lse, where, bytes;  // workspace: the kernels' own, and what the join reads
};

PrefixChoice choose(const FaPagedPrefixArgs* a) {
  PrefixChoice c{};
  const FaPagedAttnArgs& x = a->attn;
  const int64_t group = x.heads_q / x.cache.heads_kv, total = x.total;
  int64_t most[2] = {a->max_prefix_q_len, x.max_q_len};
  for (int64_t& m : most) m = (m ? std::min(m, total) : total) * group;
  c.launches = most[0] > 32 && most[1] <= 32 && tile_kernel_takes(&x) ? 2 : 1;
  c.lone_tile = most[0] <= 128;
  if (c.launches == 1) most[0] = std::max(most[0], most[1]);
  for (int i = 0; i < c.launches; ++i) {
    c.kernel[i] = choose_for_rows(&x, most[i]);
    c.kernel[i].grid = std::min(c.kernel[i].grid, +PagedWhere::kMostCtas);
    c.own[i] = c.bytes;
    c.bytes += c.kernel[i].bytes;
  }
  const int64_t rows = 2 * total * x.heads_q;
  c.whole_o = c.bytes;
  c.whole_lse = up256(c.whole_o + 4 * rows * x.cache.head_dim);
  c.where = up256(c.whole_lse + 4 * rows);
  c.bytes = up256(c.where + 4 * rows);
  return c;
}

int launch_levels(const PagedPlan& plan) {
  const bool tile = plan.rows == 0;
  switch (plan.params.head_dim) {
    case 16: return tile ? launch_levels_tile_d16(plan) : launch_levels_rows_d16(plan);
    case 32: return tile ? launch_levels_tile_d32(plan) : launch_levels_rows_d32(plan);
    case 64: return tile ? launch_levels_tile_d64(plan) : launch_levels_rows_d64(plan);
    case 128: return tile ? launch_levels_tile_d128(plan) : launch_levels_rows_d128(plan);
    default: return tile ? launch_levels_tile_d256(plan) : launch_levels_rows_d256(plan);
  }
}

// What a tile takes of an SM, relative to 200 for one of the tile kernel; 0: the two kernels do not run side by
// side but one behind the other on all SMs.  Found by trying (head_dim 128, 8 kv heads, prefixes of 8000 to
// 60,000 tokens, 16 to 128 sequences): side by side took 80 us where one behind the other took 101 for 64
// single tokens in 16 bits (8-row blocks), 99 and 127 for 4 new tokens of 48 sequences (16-row blocks), 100 and
// 118 for 8 of 32 (32-row blocks), 117 and 132 for 64 single tokens in float8; but 176 and 169 for 4 of 40 in
// float8, where the row kernel is bound by its chain and its blocks differ in time.  Other head_dims go by the same
// numbers, unmeasured; nothing but the balance depends on them.
int unit_of(const PagedPlan& plan, const PagedInfo& info, const PagedPlan& own, bool lone_tile) {
  if (own.fp8 && own.rows > 8) return 0;
  if (plan.rows == 0) return lone_tile ? 130 : 200;  // (both sides of a CTA work on a lone query tile)
  if (plan.rows > 8) return plan.rows == 16 ? 150 : 120;
  const int bytes = 2 * info.keys * plan.params.head_dim * (plan.fp8 ? 1 : 2);
  return std::max(40, bytes * (plan.fp8 ? 100 : 70) / 65536);
}

int prefix_attention(const FaPagedPrefixArgs* a, void* stream) {
  int rc = check_prefix(a);
  if (rc != FA_OK) return rc;
  const FaPagedAttnArgs x[2] = {of_prefixes(a), a->attn};
  for (int i = 0; i < 2 && rc == FA_OK; ++i) rc = check_cache(x[i].cache, x[i].dtype, x[i].total);
  if (rc != FA_OK) return rc;
  if (a->attn.total == 0 || a->attn.cache.seqs == 0) return FA_OK;
  rc = check_attn_pointers(&a->attn);
  if (rc == FA_OK) rc = check_device();
  if (rc != FA_OK) return rc;
  const PrefixChoice c = choose(a);
  if (a->attn.workspace_bytes < c.bytes) return FA_ERR_INVALID_ARG;

  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(a->attn.workspace);
  const PagedSeqs seqs[2] = {seqs_of(x[0].cache, x[0].total, x[0].dev_status),
                             seqs_of(x[1].cache, x[1].total, x[1].dev_status)};
  PagedPlan plan[2] = {};
  JoinParams j{};
  for (int i = 0; i < c.launches; ++i) {
    rc = plan_attn(&a->attn, c.kernel[i], ws + c.own[i], s, plan[i]);
    if (rc != FA_OK) return rc;
    PagedLevelParams& p = plan[i].params;
    const PagedInfo& info = c.kernel[i].info;
    p.whole_items = 0;  // (there is a join in any case)
    p.min_steps_log2 = plan[i].rows == 0 ? 2 : 1;
    p.seqs = seqs[0];
    p.own = seqs[1];
    p.lse = reinterpret_cast<float*>(ws + c.whole_lse);
    p.whole_o = reinterpret_cast<float*>(ws + c.whole_o);
    p.where = reinterpret_cast<uint32_t*>(ws + c.where);
    p.rows = a->attn.total * a->attn.heads_q;
    if (c.launches == 2) {
      p.place = i + 1;
      (i == 0 ? p.own : p.seqs).seqs = 0;
    }
    for (int k = c.launches == 2 ? i : 0; k < (c.launches == 2 ? i + 1 : 2); ++k)
      j.level[k] = JoinLevel{p.part_o, p.part_lse, seqs[k].offsets, seqs[k].seqs, info.rows, c.kernel[i].grid};
  }
  for (int i = 0; c.launches == 2 && i < 2; ++i) {
    const PagedAttnParams& p = plan[i].params;
    const PagedInfo& info = c.kernel[i].info;
    const int rows = plan[i].rows == 0 ? info.rows / 128 * p.tile_live : info.rows;
    // (short sequences cost their start more than the line counts)
    const PagedLevel v{seqs[i], rows, info.keys, p.item_cost + 2 * (plan[i].rows > 0),
                       unit_of(plan[i], info, plan[1], c.lone_tile)};
    plan[0].params.levels[i] = plan[1].params.levels[i] = v;
  }
  for (int i = 0; i < c.launches; ++i) {
    rc = launch_levels(plan[i]);
    if (rc != 0) return rc;
  }
  j.whole_o = plan[0].params.whole_o;
  j.whole_lse = plan[0].params.lse;
  j.where = plan[0].params.where;
  j.o = a->attn.o;
  j.lse = a->attn.lse;
  for (int d = 0; d < 2; ++d) j.o_stride[d] = a->attn.o_stride[d];
  j.heads_q = static_cast<int>(a->attn.heads_q);
  j.rows = static_cast<int>(plan[0].params.rows);
  // Parts are shared among threads while that leaves few enough blocks to be on the SMs at once.
  const int64_t blocks = static_cast<int64_t>(j.rows) * a->attn.cache.head_dim / kJoinThreads;
  const bool split = blocks <= 16 * c.kernel[0].grid;
  return plan[0].half ? join<__half>(j, a->attn.cache.head_dim, split, s)
                      : join<__nv_bfloat16>(j, a->attn.cache.head_dim, split, s);
}

}  // namespace
}  // namespace fa

extern "C" {

int64_t fa_paged_prefix_workspace_bytes(const FaPagedPrefixArgs* a) {
  const int rc = fa::check_prefix(a);
  return rc != FA_OK ? rc : fa::choose(a).bytes;
}

int fa_paged_prefix_sm100(const FaPagedPrefixArgs* a, void* stream) {
  return fa::prefix_attention(a, stream);
}

}  // extern "C"
