// Eviction from the paged key/value cache by accumulated attention weight (fa_paged_evict_sm100 of
// include/fa_paged_sm100.h).  Of a sequence longer than `keep` each kv head keeps its last `recent` tokens
// and, of the others, the keep - recent with the largest weights, the earlier one of two equal ones.  They
// stay in their order: rank i goes to slot i.
//
// Two launches.  paged_select_kernel finds the ranks of a (sequence, head): the weight of the last token
// that stays is found digit by digit from the top (four histograms of 8 bits), over keys that are read
// from memory once and then lie in shared memory; an ordered scan then writes the positions that stay.  A
// long sequence is shared by a cluster of up to 8 CTAs, which add their histograms up through distributed
// shared memory.  paged_move_kernel moves the rows, bound by memory.
//
// In place: slot i is written by rank i and read by a rank <= i, as rank(s) <= s.  So a CTA that goes
// through the ranks in order, a chunk at a time, may write a chunk once it has read it and all before it,
// and may read any number of chunks ahead.  CTAs that must not wait for one another take different columns
// of the rows.
#include <algorithm>

#include "fa_paged_host.h"
#include "fa_paged_launch.h"

namespace fa {
namespace {

struct EvictParams {
  PagedSeqs seqs;
  float* weights;
  int64_t weights_stride[2];  // page, head
  int heads;
  int keep, recent;
  int* kept;      // [seqs, heads, keep]
  int* new_lens;  // [seqs]
  int cached;     // keys of a CTA that fit shared memory
  // moving
  const int* to_table;
  int64_t to_stride;
  int to_cols;
  int in_place;
  void* cache[2];
  int64_t cache_stride[2][3];  // bytes
  float* scale[2];             // null: 16-bit cache
  int64_t scale_stride[2][2];
  int slices;      // column slices of a row of K or V
  int lanes_log2;  // 16-byte pieces of a slice
  int splits;      // ranges of ranks (not in place)
};

// --------------------------------------------------------------------------------- selection
constexpr int kSelectThreads = 512;
constexpr int kBins = 256;
constexpr int kMostCluster = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t x;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(x));
  return x;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t x;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(x));
  return x;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The word at shared address `addr` of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t x;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
      : "=r"(x)
      : "r"(addr), "r"(rank)
      : "memory");
  return x;
}

// Unsigned numbers in the order of floats; -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t b = w == 0.f ? 0u : __float_as_uint(w);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_key[];
  __shared__ uint32_t s_hist[kBins * 32];   // a column for each lane: no two of a warp meet
  __shared__ uint32_t s_total[2][kBins];    // read by the cluster
  __shared__ uint32_t s_count[2];           // ... keys above the threshold, keys at it
  __shared__ uint32_t s_found[2];           // digit, and how many are wanted at it
  __shared__ uint32_t s_warp[2][kSelectThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cs = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int item = blockIdx.x / cs;
  const int b = item / p.heads, head = item - b * p.heads;
  let_next_launch();
  wait_for_launch_before();
  const int n = seq_len(p.seqs, b);
  const int stay = min(n, p.keep);
  int* const kept = p.kept + static_cast<int64_t>(item) * p.keep;
  if (rank == 0 && head == 0 && tid == 0) {
    p.new_lens[b] = stay;
    if (fresh(p.seqs.kv_lens + b) != n) report(p.seqs.status, kStatusPageTable);
  }
  for (int i = stay + rank * kSelectThreads + tid; i < p.keep; i += cs * kSelectThreads) kept[i] = -1;
  if (n <= p.keep) {  // (the whole cluster)
    for (int i = rank * kSelectThreads + tid; i < n; i += cs * kSelectThreads) kept[i] = i;
    return;
  }
  const int old = n - p.recent;             // positions that may go
  const uint32_t want = p.keep - p.recent;  // and how many of them stay
  for (int i = rank * kSelectThreads + tid; i < p.recent; i += cs * kSelectThreads) kept[want + i] = old + i;
  if (want == 0) return;

  // this CTA's positions
  const int share = ((old + cs - 1) / cs + 3) & ~3;
  const int lo = min(rank * share, old), count = min(share, old - lo);
  auto from_memory = [&](int i) -> uint32_t {
    const int pos = lo + i;
    const int page = checked_page(p.seqs, page_entry(p.seqs, b, pos));
    return order_of(fresh(p.weights + page * p.weights_stride[0] + head * p.weights_stride[1] +
                          (pos & ((1 << p.seqs.page_log2) - 1))));
  };
  auto key = [&](int i) -> uint32_t { return i < p.cached ? s_key[i] : from_memory(i); };
  const int in_shared = min(count, p.cached);
#pragma unroll 4
  for (int i = tid; i < in_shared; i += kSelectThreads) s_key[i] = from_memory(i);

  uint32_t found = 0, left = want;
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    for (int i = tid; i < kBins * 32; i += kSelectThreads) s_hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < count; i += kSelectThreads) {
      const uint32_t k = key(i);
      if (pass == 0 || (k ^ found) >> (shift + 8) == 0) atomicAdd(&s_hist[(k >> shift & 255) * 32 + lane], 1u);
    }
    __syncthreads();
    if (tid < kBins) {
      uint32_t sum = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) sum += s_hist[tid * 32 + ((j + lane) & 31)];
      s_total[pass & 1][tid] = sum;
    }
    cluster_sync();
    if (warp == 0) {  // a lane for 8 bins, the highest first
      uint32_t bins[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int bin = kBins - 1 - (lane * 8 + j);
        bins[j] = 0;
        for (int c = 0; c < cs; ++c) bins[j] += ld_cluster(smem_u32(&s_total[pass & 1][bin]), c);
        sum += bins[j];
      }
      uint32_t upto = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
      }
      uint32_t before = upto - sum;
      if (before < left && left <= upto) {  // one lane
        int j = 0;
        while (before + bins[j] < left) before += bins[j++];
        s_found[0] = kBins - 1 - (lane * 8 + j);
        s_found[1] = left - before;
      }
    }
    __syncthreads();
    found |= s_found[0] << shift;
    left = s_found[1];
  }
  // `left` of the keys equal to `found` stay, the first ones, and all above it
  uint32_t above = 0, equal = 0;
  for (int i = tid; i < count; i += kSelectThreads) {
    const uint32_t k = key(i);
    above += k > found;
    equal += k == found;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    above += __shfl_xor_sync(0xffffffffu, above, d);
    equal += __shfl_xor_sync(0xffffffffu, equal, d);
  }
  if (lane == 0) {
    s_warp[0][warp] = above;
    s_warp[1][warp] = equal;
  }
  __syncthreads();
  if (tid < 2) {
    uint32_t sum = 0;
    for (int w = 0; w < kSelectThreads / 32; ++w) sum += s_warp[tid][w];
    s_count[tid] = sum;
  }
  cluster_sync();
  above = equal = 0;  // those of the CTAs before
  for (int c = 0; c < rank; ++c) {
    above += ld_cluster(smem_u32(&s_count[0]), c);
    equal += ld_cluster(smem_u32(&s_count[1]), c);
  }
  constexpr int kEach = 4;  // keys of a thread at a time
  for (int at = 0; at < count; at += kSelectThreads * kEach) {
    uint32_t k[kEach], mine = 0;  // above in the low half, equal in the high one
    const int i0 = at + tid * kEach;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      k[j] = i0 + j < count ? key(i0 + j) : 0u;
      if (i0 + j < count) mine += (k[j] > found) | (k[j] == found) << 16;
    }
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    __syncthreads();
    if (lane == 31) s_warp[0][warp] = upto;
    __syncthreads();
    uint32_t before = upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 32; ++w) {
      if (w < warp) before += s_warp[0][w];
      all += s_warp[0][w];
    }
    uint32_t a = above + (before & 0xffffu), e = equal + (before >> 16);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (i0 + j >= count) break;
      if (k[j] > found) kept[a++ + min(e, left)] = lo + i0 + j;
      else if (k[j] == found && e++ < left) kept[a + e - 1] = lo + i0 + j;
    }
    above += all & 0xffffu;
    equal += all >> 16;
  }
  cluster_sync();  // nobody reads this CTA's shared memory any more
}

// ------------------------------------------------------------------------------------ moving
constexpr int kMoveThreads = 512;
constexpr int kMoveUnroll = 4;

// One block: (sequence, head), and a column slice of K or V, or the weights and scales.
__global__ void __launch_bounds__(kMoveThreads, 2) paged_move_kernel(const __grid_constant__ EvictParams p) {
  constexpr int U = kMoveUnroll;
  const int pieces = 2 * p.slices + 1;
  const int piece = blockIdx.x % pieces, item = blockIdx.x / pieces;
  const int b = item / p.heads, head = item - b * p.heads;
  let_next_launch();
  wait_for_launch_before();
  const int n = seq_len(p.seqs, b);
  if (p.in_place && n <= p.keep) return;
  int stay = min(n, p.keep), from = 0;
  if (p.splits > 1) {  // (not in place)
    const int each = (stay + p.splits - 1) / p.splits;
    from = min(static_cast<int>(blockIdx.y) * each, stay);
    stay = min(from + each, stay);
  }
  const int* const kept = p.kept + static_cast<int64_t>(item) * p.keep;
  const int mask = (1 << p.seqs.page_log2) - 1;
  // source and destination of rank i: pages and slots; false: stays where it is, or has no place
  auto place = [&](int i, int& page, int& slot, int& to_page) -> bool {
    if (i >= stay) return false;
    const int pos = fresh(kept + i);
    if (p.in_place && pos == i) return false;
    const int col = i >> p.seqs.page_log2;
    if (static_cast<uint32_t>(pos) >= static_cast<uint32_t>(n) || col >= p.to_cols) {
      report(p.seqs.status, kStatusPageTable);
      return false;
    }
    page = page_entry(p.seqs, b, pos);
    to_page = fresh(p.to_table + b * p.to_stride + col);
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.seqs.num_pages) ||
        static_cast<uint32_t>(to_page) >= static_cast<uint32_t>(p.seqs.num_pages)) {
      report(p.seqs.status, kStatusPageTable);
      return false;
    }
    slot = pos & mask;
    return true;
  };
  if (piece < 2 * p.slices) {
    const int kv = piece / p.slices, lanes = 1 << p.lanes_log2;
    char* const cache = static_cast<char*>(p.cache[kv]) + head * p.cache_stride[kv][1] +
                        ((piece % p.slices) * lanes + (threadIdx.x & (lanes - 1))) * 16;
    const int rows = kMoveThreads >> p.lanes_log2;  // at a time
    const int r0 = from + (threadIdx.x >> p.lanes_log2);
    uint4 x[U], y[U];
    int64_t to[U], to_next[U];  // < 0: nothing to write
    auto load = [&](int at, uint4(&v)[U], int64_t(&dst)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = at + u * rows + r0 - from;
        int page, slot, to_page;
        dst[u] = -1;
        if (place(i, page, slot, to_page)) {
          v[u] = fresh(reinterpret_cast<const uint4*>(cache + page * p.cache_stride[kv][0] + slot * p.cache_stride[kv][2]));
          dst[u] = to_page * p.cache_stride[kv][0] + (i & mask) * p.cache_stride[kv][2];
        }
      }
    };
    load(from, x, to);
    for (int at = from; at < stay; at += U * rows) {
      load(at + U * rows, y, to_next);
      __syncthreads();  // the chunk has been read by all
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (to[u] >= 0) *reinterpret_cast<uint4*>(cache + to[u]) = x[u];
        x[u] = y[u];
        to[u] = to_next[u];
      }
    }
    return;
  }
  for (int at = from; at < stay; at += kMoveThreads) {
    const int i = at + threadIdx.x;
    int page, slot, to_page;
    const bool moves = place(i, page, slot, to_page);
    float w = 0.f, s[2] = {0.f, 0.f};
    if (moves) {
      w = fresh(p.weights + page * p.weights_stride[0] + head * p.weights_stride[1] + slot);
      if (p.scale[0])
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
          s[kv] = fresh(p.scale[kv] + page * p.scale_stride[kv][0] + head * p.scale_stride[kv][1] + slot);
    }
    __syncthreads();
    if (moves) {
      p.weights[to_page * p.weights_stride[0] + head * p.weights_stride[1] + (i & mask)] = w;
      if (p.scale[0])
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
          p.scale[kv][to_page * p.scale_stride[kv][0] + head * p.scale_stride[kv][1] + (i & mask)] = s[kv];
    }
  }
}

int evict(const FaPagedEvictArgs* a, void* stream) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(FaPagedEvictArgs))) return FA_ERR_INVALID_ARG;
  FaPagedCache c = a->cache;
  c.offsets = c.kv_lens;  // (there are no packed rows)
  const bool f8 = c.dtype == FA_DTYPE_FP8_E4M3;
  int rc = check_layout(c, f8 ? FA_DTYPE_BF16 : c.dtype, 0);
  if (rc != FA_OK) return rc;
  constexpr int64_t kMost = int64_t{1} << 30;
  if (a->keep < 0 || a->keep > kMost || a->recent < 0 || a->recent > a->keep) return FA_ERR_INVALID_ARG;
  if (!a->in_place && (a->to_cols < 0 || a->to_cols > kMost || a->to_cols * c.page_size > kMost))
    return FA_ERR_INVALID_ARG;
  for (int d = 0; d < 2; ++d)
    if (a->weights_stride[d] <= 0 || a->weights_stride[d] % 4) return FA_ERR_MISALIGNED;
  if (c.seqs * c.heads_kv > kMost / 64) return FA_ERR_INVALID_ARG;
  if (c.seqs == 0) return FA_OK;
  rc = check_cache(c, f8 ? FA_DTYPE_BF16 : c.dtype, 0);
  if (rc != FA_OK) return rc;
  if (!a->weights || !a->new_lens || (a->keep > 0 && !a->kept) || (!a->in_place && a->to_cols > 0 && !a->to_table))
    return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a->weights) % 16) return FA_ERR_MISALIGNED;
  rc = check_device();
  if (rc != FA_OK) return rc;

  EvictParams p{};
  p.seqs = seqs_of(c, 0, a->dev_status);
  p.weights = a->weights;
  p.heads = static_cast<int>(c.heads_kv);
  p.keep = static_cast<int>(a->keep);
  p.recent = static_cast<int>(a->recent);
  p.kept = a->kept;
  p.new_lens = a->new_lens;
  p.in_place = a->in_place ? 1 : 0;
  p.to_table = p.in_place ? c.page_table : a->to_table;
  p.to_stride = p.in_place ? c.table_stride : a->to_stride;
  p.to_cols = static_cast<int>(p.in_place ? c.table_cols : a->to_cols);
  const int eb = f8 ? 1 : 2;
  for (int i = 0; i < 2; ++i) {
    p.weights_stride[i] = a->weights_stride[i];
    p.cache[i] = i ? c.v : c.k;
    p.scale[i] = f8 ? (i ? c.v_scale : c.k_scale) : nullptr;
    for (int d = 0; d < 3; ++d) p.cache_stride[i][d] = (i ? c.v_stride : c.k_stride)[d] * eb;
    for (int d = 0; d < 2; ++d) p.scale_stride[i][d] = (i ? c.v_scale_stride : c.k_scale_stride)[d];
  }
  const int sms = sm_count_of_current();
  const int64_t items = c.seqs * c.heads_kv, capacity = c.table_cols * c.page_size;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);

  // A (sequence, head) gets more CTAs while they find an SM and have 2048 keys each.
  int cluster = 1;
  while (cluster < kMostCluster && items * cluster * 2 <= sms && capacity > 2048 * cluster) cluster *= 2;
  const int64_t share = (capacity + cluster - 1) / cluster + 4;
  p.cached = static_cast<int>(std::min<int64_t>(share, 44 * 1024));  // 176 KB, 34 KB are the kernel's own
  const int smem = p.cached * 4;
  static SmemOptIn opt_in;
  if (!opt_in(reinterpret_cast<const void*>(paged_select_kernel), 44 * 1024 * 4)) return FA_ERR_LAUNCH;
  {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(items * cluster));
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, paged_select_kernel, p) != cudaSuccess) {
      (void)cudaGetLastError();
      return FA_ERR_LAUNCH;
    }
  }
  if (p.keep == 0) return FA_OK;
  // Slices: rows whole, or in parts of at least 32 bytes while that finds SMs without work.
  const int row_bytes = static_cast<int>(c.head_dim) * eb;
  p.slices = 1;
  while (row_bytes / p.slices > 32 && items * 2 * p.slices < 2 * sms) p.slices *= 2;
  p.lanes_log2 = log2_of(row_bytes / p.slices / 16);
  p.splits = 1;
  if (!p.in_place) {
    p.slices = 1;
    p.lanes_log2 = log2_of(row_bytes / 16);
    const int64_t chunk = kMoveThreads * kMoveUnroll >> p.lanes_log2;
    p.splits = static_cast<int>(std::min<int64_t>((p.keep + 2 * chunk - 1) / (2 * chunk), 1024));
  }
  const dim3 grid(static_cast<unsigned>(items * (2 * p.slices + 1)), static_cast<unsigned>(p.splits));
  return launch_dependent(paged_move_kernel, grid, kMoveThreads, 0, s, p);
}

}  // namespace
}  // namespace fa

extern "C" {

int fa_paged_evict_sm100(const FaPagedEvictArgs* args, void* stream) { return fa::evict(args, stream); }

}  // extern "C"
