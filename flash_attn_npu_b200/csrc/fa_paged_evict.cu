// Eviction from the paged key/value cache by accumulated attention weight (fa_paged_evict_sm100 of
// include/fa_paged_sm100.h).  Of a sequence longer than `keep` each kv head keeps its last `recent` tokens
// and, of the others, the keep - recent with the largest weights, the earlier one of two equal ones.  They
// stay in their order: rank i goes to slot i.
//
// Two launches.  paged_select_kernel finds the ranks of a (sequence, head): the weight of the last token
// that stays is found digit by digit from the top (histograms of 11, 11 and 10 bits), over keys that are read
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
constexpr int kBins = 2048;
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

// THREADS: 512, or 1024 for many keys, whose histogram has four columns then (lane by lane: fewer of a warp
// meet in a word, where weights are alike).  CLUSTER: several CTAs share an item.
template <int THREADS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS) paged_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int COLS = THREADS == 1024 ? 4 : 1;
  constexpr int EACH = kBins / THREADS;  // bins of a thread
  constexpr int WARPS = THREADS / 32;
  extern __shared__ __align__(16) uint32_t s_mem[];
  uint32_t* const s_hist = s_mem;                                // [kBins][COLS]
  uint4* const s_key4 = reinterpret_cast<uint4*>(s_mem + kBins * COLS);
  const uint32_t* const s_key = s_mem + kBins * COLS;
  __shared__ __align__(16) uint32_t s_total[2][kBins];  // read by the cluster
  __shared__ uint32_t s_count[2];           // ... keys above the threshold, keys at it
  __shared__ uint32_t s_found[3];           // digit, how many are wanted at it, and how many there are
  __shared__ uint32_t s_warp[2][WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cs = CLUSTER ? static_cast<int>(cluster_size()) : 1;
  const int rank = CLUSTER ? static_cast<int>(cluster_rank()) : 0;
  auto sync_all = [&]() {
    if (CLUSTER) cluster_sync();
    else __syncthreads();
  };
  auto of_cta = [&](const uint32_t& x, int c) -> uint32_t { return CLUSTER ? ld_cluster(smem_u32(&x), c) : x; };
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
  for (int i = stay + rank * THREADS + tid; i < p.keep; i += cs * THREADS) kept[i] = -1;
  if (n <= p.keep) {  // (the whole cluster)
    for (int i = rank * THREADS + tid; i < n; i += cs * THREADS) kept[i] = i;
    return;
  }
  const int old = n - p.recent;             // positions that may go
  const uint32_t want = p.keep - p.recent;  // and how many of them stay
  for (int i = rank * THREADS + tid; i < p.recent; i += cs * THREADS) kept[want + i] = old + i;
  if (want == 0) return;

  // this CTA's positions, four at a time: they lie in one page, 16 bytes together
  const int share = ((old + cs - 1) / cs + 3) & ~3;
  const int lo = min(rank * share, old), count = min(share, old - lo);
  const int mask = (1 << p.seqs.page_log2) - 1;
  auto from_memory = [&](int i4) -> uint4 {
    const int pos = lo + 4 * i4;
    const int page = checked_page(p.seqs, page_entry(p.seqs, b, pos));
    const float4 x = fresh(reinterpret_cast<const float4*>(p.weights + page * p.weights_stride[0] +
                                                           head * p.weights_stride[1] + (pos & mask)));
    return make_uint4(order_of(x.x), order_of(x.y), order_of(x.z), order_of(x.w));
  };
  const int count4 = (count + 3) / 4, cached4 = min(count4, p.cached / 4);
  auto keys = [&](int i4) -> uint4 { return i4 < cached4 ? s_key4[i4] : from_memory(i4); };
#pragma unroll 4
  for (int i = tid; i < cached4; i += THREADS) s_key4[i] = from_memory(i);

  // A key stays if its upper digits are above `found`, and of the keys that have them equal the first `left`.
  uint32_t found = 0, left = want;
  int shift = 32, turn = 0;
  do {  // digits of 11, 11 and 10 bits
    const int bits = min(shift, 11);
    const int above_bits = shift;
    shift -= bits;
    turn ^= 1;
    for (int i = tid; i < kBins * COLS / 4; i += THREADS) reinterpret_cast<uint4*>(s_hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i = tid; i < count4; i += THREADS) {
      const uint4 k4 = keys(i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t k = (&k4.x)[j];
        if (4 * i + j < count && (above_bits == 32 || (k ^ found) >> above_bits == 0))
          atomicAdd(&s_hist[(k >> shift & ((1u << bits) - 1)) * COLS + lane % COLS], 1u);
      }
    }
    __syncthreads();
    // a thread's bins, the highest first: EACH of them below bin `top`
    const int top = kBins - 1 - tid * EACH;
    uint32_t bins[EACH], sum = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if constexpr (COLS == 4) {
        const uint4 x = reinterpret_cast<const uint4*>(s_hist)[top - j];
        bins[j] = x.x + x.y + x.z + x.w;
      } else {
        bins[j] = s_hist[top - j];
      }
      if (CLUSTER) s_total[turn][top - j] = bins[j];
    }
    if (CLUSTER) {
      cluster_sync();
#pragma unroll
      for (int j = 0; j < EACH; ++j)
        for (int c = 0; c < cs; ++c)
          if (c != rank) bins[j] += of_cta(s_total[turn][top - j], c);
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += bins[j];
    uint32_t upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 31) s_warp[0][warp] = upto;
    __syncthreads();
    uint32_t before = upto - sum;
#pragma unroll
    for (int x = 0; x < WARPS; ++x) before += x < warp ? s_warp[0][x] : 0;
    if (before < left && left <= before + sum) {  // one thread
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        if (before < left && left <= before + bins[j]) {
          s_found[0] = top - j;
          s_found[1] = left - before;
          s_found[2] = bins[j];
        }
        before += bins[j];
      }
    }
    __syncthreads();
    found |= s_found[0] << shift;
    left = s_found[1];
  } while (shift > 0 && left < s_found[2]);  // (all of a bin stay: its lower digits do not matter)
  found >>= shift;
  uint32_t above = 0, equal = 0;
  if (CLUSTER) {  // this CTA's numbers of them, for those behind it
    for (int i = tid; i < count4; i += THREADS) {
      const uint4 k4 = keys(i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t k = (&k4.x)[j] >> shift;
        above += 4 * i + j < count && k > found;
        equal += 4 * i + j < count && k == found;
      }
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
      for (int w = 0; w < WARPS; ++w) sum += s_warp[tid][w];
      s_count[tid] = sum;
    }
    cluster_sync();
  }
  above = equal = 0;  // those of the CTAs before
  for (int c = 0; c < rank; ++c) {
    above += of_cta(s_count[0], c);
    equal += of_cta(s_count[1], c);
  }
  constexpr int kEach = 4;  // keys of a thread at a time
  for (int at = 0; at < count; at += THREADS * kEach) {
    uint32_t k[kEach], mine = 0;  // above in the low half, equal in the high one
    const int i0 = at + tid * kEach;
    const uint4 k4 = i0 < count ? keys(i0 / 4) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      k[j] = (&k4.x)[j] >> shift;
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
    for (int w = 0; w < WARPS; ++w) {
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
  if (CLUSTER) cluster_sync();  // nobody reads this CTA's shared memory any more
}

// ------------------------------------------------------------------------------------ moving
constexpr int kMoveThreads = 512;
constexpr int kMoveUnroll = 4;
constexpr int kMostRows = kMoveThreads * kMoveUnroll / 2;  // of a chunk (rows of 16 bytes: half of what they could be)

// One block: (sequence, head), and a column slice of K or V, or the weights and scales.
//
// A chunk's ranks go through four stages, one turn of the loop each, so that no turn waits for more than one
// load: positions, pages, rows into registers, rows into their places.  Positions and pages are looked up
// once for a row and go through shared memory to the threads that share it.
__global__ void __launch_bounds__(kMoveThreads, 2) paged_move_kernel(const __grid_constant__ EvictParams p) {
  constexpr int U = kMoveUnroll;
  constexpr int EACH = kMostRows / kMoveThreads;  // rows that a thread looks up
  __shared__ int64_t s_from[3][kMostRows];        // bytes from the head's first; < 0: stays, or has no place
  __shared__ int s_to[3][kMostRows];              // page
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
  if (from >= stay) return;
  const int* const kept = p.kept + static_cast<int64_t>(item) * p.keep;
  const int mask = (1 << p.seqs.page_log2) - 1;
  // Position of rank i, not looked at yet (a stage may not wait for its own loads); and what it says: -1, the
  // rank stays where it is.
  auto position = [&](int i) -> int { return i < stay ? fresh(kept + i) : -1; };
  auto moving = [&](int pos, int i) -> int {
    if (i >= stay || (p.in_place && pos == i)) return -1;
    if (static_cast<uint32_t>(pos) < static_cast<uint32_t>(n)) return pos;
    report(p.seqs.status, kStatusPageTable);
    return -1;
  };
  // page that rank i goes to, or -1
  auto page_to = [&](int i) -> int {
    const int col = i >> p.seqs.page_log2;
    return col < p.to_cols ? fresh(p.to_table + b * p.to_stride + col) : -1;
  };
  auto is_page = [&](int page) -> bool {
    if (static_cast<uint32_t>(page) < static_cast<uint32_t>(p.seqs.num_pages)) return true;
    report(p.seqs.status, kStatusPageTable);
    return false;
  };
  if (piece < 2 * p.slices) {
    const int kv = piece / p.slices, lanes = 1 << p.lanes_log2;
    const int64_t st_page = p.cache_stride[kv][0], st_row = p.cache_stride[kv][2];
    char* const cache = static_cast<char*>(p.cache[kv]) + head * p.cache_stride[kv][1] +
                        ((piece % p.slices) * lanes + (threadIdx.x & (lanes - 1))) * 16;
    const int step = kMoveThreads >> p.lanes_log2;  // rows that the block takes at a time
    const int rows = min(U * step, kMostRows);      // of a chunk
    const int r0 = threadIdx.x >> p.lanes_log2;
    const int tid = threadIdx.x;
    int pos[EACH], page[EACH], to[EACH], pos_of[EACH];
    auto positions = [&](int at) {
#pragma unroll
      for (int e = 0; e < EACH; ++e)
        pos[e] = tid + e * kMoveThreads < rows ? position(at + tid + e * kMoveThreads) : -1;
    };
    auto pages = [&](int at) {
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = at + tid + e * kMoveThreads;
        pos_of[e] = tid + e * kMoveThreads < rows ? moving(pos[e], i) : -1;
        page[e] = to[e] = -1;
        if (pos_of[e] >= 0) {
          page[e] = page_entry(p.seqs, b, pos_of[e]);
          to[e] = page_to(i);
        }
      }
    };
    auto publish = [&](int slot) {
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int r = tid + e * kMoveThreads;
        if (r >= rows) continue;
        const bool moves = pos_of[e] >= 0 && is_page(page[e]) && is_page(to[e]);
        s_from[slot][r] = moves ? page[e] * st_page + (pos_of[e] & mask) * st_row : -1;
        s_to[slot][r] = to[e];
      }
    };
    uint4 x[U], y[U];
    auto load = [&](int slot, uint4(&v)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * step;
        if (r < rows && s_from[slot][r] >= 0) v[u] = fresh(reinterpret_cast<const uint4*>(cache + s_from[slot][r]));
      }
    };
    positions(from);
    pages(from);
    publish(0);
    positions(from + rows);
    pages(from + rows);
    positions(from + 2 * rows);
    __syncthreads();
    load(0, x);
    int slot = 0;  // of the chunk that is written in this turn
    auto turn = [&](int at, uint4(&now)[U], uint4(&then)[U]) {
      const int next = slot == 2 ? 0 : slot + 1;
      publish(next);
      pages(at + 2 * rows);
      positions(at + 3 * rows);
      __syncthreads();  // the next chunk's places are there, and this one has been read by all
      load(next, then);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * step;
        if (r < rows && s_from[slot][r] >= 0)
          *reinterpret_cast<uint4*>(cache + s_to[slot][r] * st_page + ((at + r) & mask) * st_row) = now[u];
      }
      slot = next;
    };
    for (int at = from; at < stay; at += 2 * rows) {
      turn(at, x, y);
      if (at + rows < stay) turn(at + rows, y, x);
    }
    return;
  }
  // The weights and scales: a float each, eight ranks to a thread at a time.
  constexpr int M = 8;
  for (int at = from; at < stay; at += M * kMoveThreads) {
    int pos[M], page[M], to[M];
    float w[M], s[2][M];
#pragma unroll
    for (int e = 0; e < M; ++e) pos[e] = position(at + threadIdx.x + e * kMoveThreads);
#pragma unroll
    for (int e = 0; e < M; ++e) {
      pos[e] = moving(pos[e], at + threadIdx.x + e * kMoveThreads);
      page[e] = to[e] = 0;
      if (pos[e] >= 0) {
        page[e] = page_entry(p.seqs, b, pos[e]);
        to[e] = page_to(at + threadIdx.x + e * kMoveThreads);
      }
    }
#pragma unroll
    for (int e = 0; e < M; ++e) {
      if (pos[e] < 0) continue;
      if (!is_page(page[e]) || !is_page(to[e])) {
        pos[e] = -1;
        continue;
      }
      const int slot = pos[e] & mask;
      w[e] = fresh(p.weights + page[e] * p.weights_stride[0] + head * p.weights_stride[1] + slot);
      if (p.scale[0])
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
          s[kv][e] = fresh(p.scale[kv] + page[e] * p.scale_stride[kv][0] + head * p.scale_stride[kv][1] + slot);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < M; ++e) {
      if (pos[e] < 0) continue;
      const int slot = (at + threadIdx.x + e * kMoveThreads) & mask;
      p.weights[to[e] * p.weights_stride[0] + head * p.weights_stride[1] + slot] = w[e];
      if (p.scale[0])
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
          p.scale[kv][to[e] * p.scale_stride[kv][0] + head * p.scale_stride[kv][1] + slot] = s[kv][e];
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

  // A (sequence, head) gets more CTAs while all of them find a place and have 2048 keys each.
  int cluster = 1;
  while (cluster < kMostCluster && items * cluster * 2 <= 2 * sms && capacity > 2048 * cluster) cluster *= 2;
  const int64_t share = ((capacity + cluster - 1) / cluster + 3) / 4 * 4 + 4;
  const bool many = share > 8192;
  const int cols = many ? 4 : 1, threads = many ? 1024 : 512;
  constexpr int kMostBytes = 200 * 1024;  // (16 KB more are the kernel's own)
  p.cached = static_cast<int>(std::min<int64_t>(share, (kMostBytes - 4 * kBins * cols) / 4));
  const int smem = 4 * (p.cached + kBins * cols);
  const auto kernel = cluster > 1 ? (many ? paged_select_kernel<1024, true> : paged_select_kernel<512, true>)
                                  : (many ? paged_select_kernel<1024, false> : paged_select_kernel<512, false>);
  static SmemOptIn opt_in[4];
  if (!opt_in[2 * (cluster > 1) + many](reinterpret_cast<const void*>(kernel), kMostBytes)) return FA_ERR_LAUNCH;
  {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(items * cluster));
    cfg.blockDim = dim3(threads);
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
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
      (void)cudaGetLastError();
      return FA_ERR_LAUNCH;
    }
  }
  if (p.keep == 0) return FA_OK;
  // Slices: rows whole, or in parts of at least 32 bytes while that finds SMs without work.
  const int row_bytes = static_cast<int>(c.head_dim) * eb;
  p.slices = 1;
  while (row_bytes / p.slices > 32 && items * 2 * p.slices < sms) p.slices *= 2;
  p.lanes_log2 = log2_of(row_bytes / p.slices / 16);
  p.splits = 1;
  if (!p.in_place) {
    p.slices = 1;
    p.lanes_log2 = log2_of(row_bytes / 16);
    // ranges of ranks while there are SMs without a pair of blocks: a block's start costs three latencies
    const int64_t chunk = kMoveThreads * kMoveUnroll >> p.lanes_log2;
    p.splits = static_cast<int>(
        std::max<int64_t>(1, std::min({(2 * sms + 2 * items - 1) / (2 * items), (p.keep + chunk - 1) / chunk, int64_t{1024}})));
  }
  const dim3 grid(static_cast<unsigned>(items * (2 * p.slices + 1)), static_cast<unsigned>(p.splits));
  return launch_dependent(paged_move_kernel, grid, kMoveThreads, 0, s, p);
}

}  // namespace
}  // namespace fa

extern "C" {

int fa_paged_evict_sm100(const FaPagedEvictArgs* args, void* stream) { return fa::evict(args, stream); }

}  // extern "C"
