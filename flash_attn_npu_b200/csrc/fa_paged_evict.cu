// Eviction from the paged key/value cache by accumulated attention weight (fa_paged_evict_sm100 of
// include/fa_paged_sm100.h).  Of a sequence longer than `keep` each kv head keeps its last `recent` tokens
// and, of the others, the keep - recent with the largest weights, the earlier one of two equal ones.  They
// stay in their order: rank i goes to slot i.
//
// Two launches.  paged_select_kernel finds the ranks of a (sequence, head): the weight of the last token
// that stays is found digit by digit from the top (histograms of 11, 11 and 10 bits), over keys that are read
// from memory once and then lie in shared memory; an ordered scan then writes the positions that stay.  A
// long sequence is shared by a cluster of up to 16 CTAs, which add their histograms up through distributed
// shared memory.  paged_move_kernel moves the rows, bound by memory.
//
// In place: slot i is written by rank i and read by rank(i) <= i.  A block that goes through the ranks in order,
// a chunk at a time, may write a chunk once it has read it and all before it, and may read any number of chunks
// ahead.  Where there are too few such blocks, a block moves one chunk of ranks: it reads
// them into registers, says so (a flag for each chunk), and writes them once all chunks before it have been
// read.  Blocks take their chunks in the order of a ticket and none waits before it has said so, so whatever a
// block waits for is already being read.
//
// Measured: 16 sequences cut from 576 to 512 tokens (8 heads x 128, 16 bits) 20 us; 48 of 800 to 6000 cut to 1024
// (float8) 16 us of selecting and 37 of moving; one of 131,067 cut to 40,000 (4 heads) 26 and 57.  Selecting is
// a few dependent passes; moving in order reaches 47 % of the memory's nominal rate, by chunks 25 %, as a
// block writes only once all chunks before its own have been read.
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
  int lanes_log2;   // 16-byte pieces of a row of K or V
  int rows;         // of a chunk of K or V
  int chunks[2];    // of K and of V; of the weights and scales
  uint32_t* flags;  // [seqs * heads][2 * chunks[0] + chunks[1]]: the chunk has been read
  uint32_t* ticket;
};

// --------------------------------------------------------------------------------- selection
constexpr int kBins = 2048;
constexpr int kMostCluster = 16;

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
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 2 : 3) paged_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int COLS = THREADS == 1024 ? 4 : 1;
  constexpr int EACH = kBins / THREADS;  // bins of a thread
  constexpr int WARPS = THREADS / 32;
  extern __shared__ __align__(16) uint32_t s_mem[];
  uint32_t* const s_hist = s_mem;                                // [kBins][COLS]
  uint4* const s_key4 = reinterpret_cast<uint4*>(s_mem + kBins * COLS);
  __shared__ uint32_t s_own[CLUSTER ? kBins : 1], s_total[CLUSTER ? kBins : 1];  // read by the cluster
  __shared__ uint32_t s_count[2];           // ... keys above the threshold, keys at it
  __shared__ uint32_t s_found[3];           // digit, how many are wanted at it, and how many there are
  __shared__ uint32_t s_warp[2][WARPS];
  __shared__ uint32_t s_len, s_differ;      // the sequence's length as this CTA has read it; others have another
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
  // One thread reads the length, and the CTAs of a cluster compare theirs: what threads do together must not
  // come apart where something changes the lengths meanwhile, though the call forbids it.
  if (tid == 0) {
    s_len = seq_len(p.seqs, b);
    s_differ = 0;
  }
  __syncthreads();
  const int n = s_len;
  const int stay = min(n, p.keep);
  int* const kept = p.kept + static_cast<int64_t>(item) * p.keep;
  if (rank == 0 && head == 0 && tid == 0) {
    p.new_lens[b] = stay;
    // (a rank behind the last column that receives is in no chunk where a chunk ends there: nothing else says so)
    if (fresh(p.seqs.kv_lens + b) != n || stay > static_cast<int64_t>(p.to_cols) << p.seqs.page_log2)
      report(p.seqs.status, kStatusPageTable);
  }
  if (p.flags && rank == 0) {
    const int units = 2 * p.chunks[0] + p.chunks[1];
    for (int i = tid; i < units; i += THREADS) p.flags[static_cast<int64_t>(item) * units + i] = 0;
    if (blockIdx.x == 0 && tid == 0) *p.ticket = 0;
  }
  for (int i = stay + rank * THREADS + tid; i < p.keep; i += cs * THREADS) kept[i] = -1;
  if (n <= p.keep) {  // (the whole cluster)
    for (int i = rank * THREADS + tid; i < n; i += cs * THREADS) kept[i] = i;
    if (CLUSTER && p.keep > p.recent) {  // (the barriers behind which the others compare)
      cluster_sync();
      cluster_sync();
    }
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
  int shift = 32;
  uint32_t above = 0, equal = 0;  // of this thread's bins: keys of the CTA above and at the digits found
  // Sum over the warps before this one, and over all, of what lane 31 of each holds.
  auto scan_warps = [&](uint32_t last, uint32_t& all) -> uint32_t {
    __syncthreads();
    if (lane == 31) s_warp[0][warp] = last;
    __syncthreads();
    uint32_t v = lane < WARPS ? s_warp[0][lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += u;
    }
    all = __shfl_sync(0xffffffffu, v, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, v, (warp + 31) & 31);
    return warp == 0 ? 0u : before;
  };
  bool differ = false;
  do {  // digits of 11, 11 and 10 bits
    const int bits = min(shift, 11);
    const int above_bits = shift;
    shift -= bits;
    for (int i = tid; i < kBins * COLS / 4; i += THREADS) reinterpret_cast<uint4*>(s_hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (tid == 0) {  // where no bin is found (weights that change meanwhile): all CTAs end alike
      s_found[0] = s_found[2] = 0;
      s_found[1] = left;
    }
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
    uint32_t bins[EACH], own[EACH], sum = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if constexpr (COLS == 4) {
        const uint4 x = reinterpret_cast<const uint4*>(s_hist)[top - j];
        bins[j] = x.x + x.y + x.z + x.w;
      } else {
        bins[j] = s_hist[top - j];
      }
      own[j] = bins[j];
      if (CLUSTER) s_own[top - j] = bins[j];
    }
    if (CLUSTER) {
      // a CTA adds up a slice of the bins, and all read the slices: all of every CTA's would be cs times as much
      const int slice = kBins / cs;
      cluster_sync();
      for (int i = tid; i < slice; i += THREADS) {
        uint32_t all = 0;
        for (int c = 0; c < cs; ++c) all += of_cta(s_own[rank * slice + i], c);
        s_total[rank * slice + i] = all;
      }
      if (above_bits == 32 && tid < cs && of_cta(s_len, tid) != n) s_differ = 1;
      cluster_sync();
      if (above_bits == 32 && s_differ) {  // (all CTAs see it)
        differ = true;
        break;
      }
#pragma unroll
      for (int j = 0; j < EACH; ++j) bins[j] = of_cta(s_total[top - j], (top - j) / slice);
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += bins[j];
    uint32_t upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    uint32_t all;
    uint32_t before = upto - sum + scan_warps(upto, all);
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
#pragma unroll
    for (int j = 0; CLUSTER && j < EACH; ++j) {
      above += top - j > static_cast<int>(s_found[0]) ? own[j] : 0;
      equal = top - j == static_cast<int>(s_found[0]) ? own[j] : j == 0 ? 0 : equal;
    }
  } while (shift > 0 && left < s_found[2]);  // (all of a bin stay: its lower digits do not matter)
  if (CLUSTER && differ) {
    if (tid == 0) report(p.seqs.status, kStatusPageTable);
    return;
  }
  found >>= shift;
  if (CLUSTER) {  // this CTA's numbers, for those behind it
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      above += __shfl_xor_sync(0xffffffffu, above, d);
      equal += __shfl_xor_sync(0xffffffffu, equal, d);
    }
    __syncthreads();
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
  constexpr int kEach = 8;  // keys of a thread at a time
  for (int at = 0; at < count; at += THREADS * kEach) {
    uint32_t k[kEach], mine = 0;  // above in the low half, equal in the high one
    const int i0 = at + tid * kEach;
    uint4 k4[kEach / 4];
#pragma unroll
    for (int j = 0; j < kEach / 4; ++j)
      k4[j] = i0 + 4 * j < count ? keys(i0 / 4 + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      k[j] = (&k4[j / 4].x)[j % 4] >> shift;
      if (i0 + j < count) mine += (k[j] > found) | (k[j] == found) << 16;
    }
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    uint32_t all;
    const uint32_t before = upto - mine + scan_warps(upto, all);
    uint32_t a = above + (before & 0xffffu), e = equal + (before >> 16);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (i0 + j >= count) break;
      uint32_t to = want;  // (weights that change meanwhile may leave more than there is place for)
      if (k[j] > found) to = a++ + min(e, left);
      else if (k[j] == found && e++ < left) to = a + e - 1;
      if (to < want) kept[to] = lo + i0 + j;
    }
    above += all & 0xffffu;
    equal += all >> 16;
  }
  if (CLUSTER) cluster_sync();  // nobody reads this CTA's shared memory any more
}

// ------------------------------------------------------------------------------------ moving
constexpr int kMoveThreads = 512;
constexpr int kMoveUnroll = 4;                            // 16-byte pieces of a thread
constexpr int kMoveRows = kMoveThreads * kMoveUnroll;     // of the smallest rows: the most of a chunk
constexpr int kMetaUnroll = 4;                            // ranks of a thread, of the weights and scales

// One block moves one chunk of ranks of a (sequence, head): of K, of V, or of the weights and scales.
__global__ void __launch_bounds__(kMoveThreads, 3) paged_move_kernel(const __grid_constant__ EvictParams p) {
  constexpr int U = kMoveUnroll, M = kMetaUnroll;
  __shared__ int64_t s_from[kMoveRows];  // bytes from the head's first; < 0: stays, or has no place
  __shared__ int s_to[kMoveRows];        // page
  __shared__ uint32_t s_unit;
  __shared__ int s_gave_up;
  const int tid = threadIdx.x;
  const int units = 2 * p.chunks[0] + p.chunks[1];
  let_next_launch();
  wait_for_launch_before();
  if (tid == 0) {
    s_unit = p.in_place ? atomicAdd(p.ticket, 1u) : blockIdx.x;
    s_gave_up = 0;
  }
  __syncthreads();
  const int item = s_unit / units, unit = s_unit - item * units;
  const int kind = min(unit / p.chunks[0], 2), chunk = unit - kind * p.chunks[0];
  const int b = item / p.heads, head = item - b * p.heads;
  const int n = seq_len(p.seqs, b);
  const int rows = kind < 2 ? p.rows : M * kMoveThreads;
  const int at = chunk * rows, stay = min(n, p.keep);
  if (at >= stay || (p.in_place && n <= p.keep)) return;
  const int* const kept = p.kept + static_cast<int64_t>(item) * p.keep;
  const int mask = (1 << p.seqs.page_log2) - 1;
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
  // Rank i's position, its page, and the page it goes to; false: it stays where it is, or has no place.
  auto place = [&](int i, int& pos, int& page, int& to) -> bool {
    if (i >= stay) return false;
    pos = fresh(kept + i);
    if (p.in_place && pos == i) return false;
    if (static_cast<uint32_t>(pos) >= static_cast<uint32_t>(n)) {
      report(p.seqs.status, kStatusPageTable);
      return false;
    }
    page = page_entry(p.seqs, b, pos);
    to = page_to(i);
    return is_page(page) && is_page(to);
  };
  // Says that this chunk has been read, and waits until all before it have been: false if that took too long.
  // `seen` depends on all that the thread has read, so the barrier is behind the reads themselves.
  auto read_by_all = [&](bool seen) -> bool {
    __syncthreads_or(seen);
    if (!p.in_place) return true;
    uint32_t* const flags = p.flags + static_cast<int64_t>(item) * units + kind * p.chunks[0];
    // One warp speaks for the block (a fence by every thread would wait for everybody's stores).
    if (tid == 0)
      asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flags + chunk), "r"(1u) : "memory");
    if (tid < 32) {
      uint64_t t0 = 0;
      for (int c = tid; c < chunk; c += 32) {
        uint32_t read = 0;
        while (true) {
          asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(read) : "l"(flags + c) : "memory");
          if (read) break;
          const uint64_t t = globaltimer_ns();
          if (t0 == 0) t0 = t;
          if (t - t0 >= FA_WAIT_TIMEOUT_NS) {
            report(p.seqs.status, kStatusTimeout);
            s_gave_up = 1;
            break;
          }
        }
        if (!read) break;
      }
      asm volatile("fence.acq_rel.gpu;" ::: "memory");  // (the flags were seen before anything is written)
    }
    __syncthreads();
    return s_gave_up == 0;
  };
  if (kind < 2) {
    const int lanes = 1 << p.lanes_log2;
    const int64_t st_page = p.cache_stride[kind][0], st_row = p.cache_stride[kind][2];
    char* const cache =
        static_cast<char*>(p.cache[kind]) + head * p.cache_stride[kind][1] + (tid & (lanes - 1)) * 16;
    for (int r = tid; r < rows; r += kMoveThreads) {
      int pos, page, to = 0;
      const bool moves = place(at + r, pos, page, to);
      s_from[r] = moves ? page * st_page + (pos & mask) * st_row : -1;
      s_to[r] = to;
    }
    __syncthreads();
    const int step = kMoveThreads >> p.lanes_log2, r0 = tid >> p.lanes_log2;
    uint4 x[U];
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = make_uint4(0, 0, 0, 0);
      const int64_t from = s_from[r0 + u * step];
      if (from >= 0) x[u] = fresh(reinterpret_cast<const uint4*>(cache + from));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) any |= x[u].x | x[u].y | x[u].z | x[u].w;
    if (!read_by_all(any != 0)) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step;
      if (s_from[r] >= 0)
        *reinterpret_cast<uint4*>(cache + s_to[r] * st_page + ((at + r) & mask) * st_row) = x[u];
    }
    return;
  }
  int to[M];
  float w[M], sc[2][M];
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < M; ++e) {
    int pos, page;
    w[e] = sc[0][e] = sc[1][e] = 0.f;
    if (!place(at + tid + e * kMoveThreads, pos, page, to[e])) {
      to[e] = -1;
      continue;
    }
    const int slot = pos & mask;
    w[e] = fresh(p.weights + page * p.weights_stride[0] + head * p.weights_stride[1] + slot);
    if (p.scale[0])
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        sc[kv][e] = fresh(p.scale[kv] + page * p.scale_stride[kv][0] + head * p.scale_stride[kv][1] + slot);
  }
#pragma unroll
  for (int e = 0; e < M; ++e) any |= __float_as_uint(w[e]) | __float_as_uint(sc[0][e]) | __float_as_uint(sc[1][e]);
  if (!read_by_all(any != 0)) return;
#pragma unroll
  for (int e = 0; e < M; ++e) {
    if (to[e] < 0) continue;
    const int slot = (at + tid + e * kMoveThreads) & mask;
    p.weights[to[e] * p.weights_stride[0] + head * p.weights_stride[1] + slot] = w[e];
    if (p.scale[0])
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        p.scale[kv][to[e] * p.scale_stride[kv][0] + head * p.scale_stride[kv][1] + slot] = sc[kv][e];
  }
}

// In place, where there are (sequence, head) pairs enough: one block moves all of K, of V, or of the weights
// and scales, chunk by chunk in order, so it needs no flags.
//
// A chunk's ranks go through four stages, one turn of the loop each, so that no turn waits for more than one
// load: positions, pages, rows into registers, rows into their places.  Positions and pages are looked up
// once for a row and go through shared memory to the threads that share it.
// EACH: rows that a thread looks up, 1 where rows have 64 bytes at least.
template <int EACH>
__global__ void __launch_bounds__(kMoveThreads, 2) paged_move_in_order_kernel(const __grid_constant__ EvictParams p) {
  constexpr int U = kMoveUnroll;
  constexpr int ROWS = EACH * kMoveThreads;   // (rows of 16 bytes: half of what they could be)
  __shared__ int64_t s_from[3][ROWS];         // bytes from the head's first; < 0: stays, or has no place
  __shared__ int s_to[3][ROWS];               // page
  const int kind = blockIdx.x % 3, item = blockIdx.x / 3;
  const int b = item / p.heads, head = item - b * p.heads;
  let_next_launch();
  wait_for_launch_before();
  const int n = seq_len(p.seqs, b);
  if (n <= p.keep) return;
  const int stay = p.keep;
  const int* const kept = p.kept + static_cast<int64_t>(item) * p.keep;
  const int mask = (1 << p.seqs.page_log2) - 1;
  // Position of rank i, not looked at yet (a stage may not wait for its own loads); and what it says: -1, the
  // rank stays where it is.
  auto position = [&](int i) -> int { return i < stay ? fresh(kept + i) : -1; };
  auto moving = [&](int pos, int i) -> int {
    if (i >= stay || pos == i) return -1;
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
  if (kind < 2) {
    const int lanes = 1 << p.lanes_log2;
    const int64_t st_page = p.cache_stride[kind][0], st_row = p.cache_stride[kind][2];
    char* const cache = static_cast<char*>(p.cache[kind]) + head * p.cache_stride[kind][1] +
                        (threadIdx.x & (lanes - 1)) * 16;
    const int step = kMoveThreads >> p.lanes_log2;  // rows that the block takes at a time
    const int rows = min(U * step, ROWS);      // of a chunk
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
    positions(0);
    pages(0);
    publish(0);
    positions(rows);
    pages(rows);
    positions(2 * rows);
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
    for (int at = 0; at < stay; at += 2 * rows) {
      turn(at, x, y);
      if (at + rows < stay) turn(at + rows, y, x);
    }
    return;
  }
  // The weights and scales: a float each, eight ranks to a thread at a time.
  constexpr int M = 8;
  for (int at = 0; at < stay; at += M * kMoveThreads) {
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

// The division of the moving among blocks, and the workspace: a ticket, a flag for each chunk.
struct EvictChoice {
  int lanes_log2, rows, chunks[2];
  int64_t blocks, bytes;
  bool in_order;
};

EvictChoice choose(const FaPagedEvictArgs* a) {
  EvictChoice c{};
  const int64_t capacity = (a->in_place ? a->cache.table_cols : a->to_cols) * a->cache.page_size;
  const int64_t most = std::max<int64_t>(1, std::min(a->keep, capacity));
  const int row_bytes = static_cast<int>(a->cache.head_dim) * (a->cache.dtype == FA_DTYPE_FP8_E4M3 ? 1 : 2);
  c.lanes_log2 = log2_of(row_bytes / 16);
  c.rows = kMoveRows >> c.lanes_log2;
  c.chunks[0] = static_cast<int>((most + c.rows - 1) / c.rows);
  c.chunks[1] = static_cast<int>((most + kMetaUnroll * kMoveThreads - 1) / (kMetaUnroll * kMoveThreads));
  c.blocks = a->cache.seqs * a->cache.heads_kv * (2 * c.chunks[0] + c.chunks[1]);
  // In order where that gives every SM a block.  There are fewer latencies to a byte then: moving took 13 us and
  // 24 with a block a chunk for 16 sequences of 8 heads cut to 512 tokens (head_dim 128, 16 bits), 37 and 65
  // for 48 in float8 cut to 1024; one sequence of 4 heads cut to 40,000 takes 60 us with a block a chunk, and took
  // 115 in order with the columns dealt out to 16 blocks a head.  (Between 4 and 128 heads neither was measured.)
  const int64_t items = a->cache.seqs * a->cache.heads_kv;
  c.in_order = a->in_place && 2 * items >= sm_count_of_current();
  if (c.in_order) c.blocks = 3 * items;
  c.bytes = 256 + up256(a->in_place && !c.in_order ? 4 * c.blocks : 0);
  return c;
}

int check_evict(const FaPagedEvictArgs* a) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(FaPagedEvictArgs))) return FA_ERR_INVALID_ARG;
  FaPagedCache c = a->cache;
  const bool f8 = c.dtype == FA_DTYPE_FP8_E4M3;
  const int rc = check_layout(c, f8 ? FA_DTYPE_BF16 : c.dtype, 0);
  if (rc != FA_OK) return rc;
  constexpr int64_t kMost = int64_t{1} << 30;
  if (a->keep < 0 || a->keep > kMost || a->recent < 0 || a->recent > a->keep) return FA_ERR_INVALID_ARG;
  if (!a->in_place && (a->to_cols < 0 || a->to_cols > kMost || a->to_cols * c.page_size > kMost))
    return FA_ERR_INVALID_ARG;
  for (int d = 0; d < 2; ++d)
    if (a->weights_stride[d] <= 0 || a->weights_stride[d] % 4) return FA_ERR_MISALIGNED;
  if (c.seqs * c.heads_kv > kMost / 64 || choose(a).blocks > INT32_MAX) return FA_ERR_INVALID_ARG;
  return FA_OK;
}

constexpr int kMostBytes = 200 * 1024;  // of a selecting block's shared memory (16 KB more are the kernel's own)

// Whether clusters of 16 selecting blocks find a place on the current device (more than 8 have to be asked for).
bool large_clusters() {
  static std::atomic<int> known[16] = {};  // 1: yes, 2: no
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) return false;
  int is = known[dev].load(std::memory_order_acquire);
  if (is == 0) {
    const auto kernel = paged_select_kernel<1024, true>;
    const void* const fn = reinterpret_cast<const void*>(kernel);
    int n = 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = kMostBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 16;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool ok = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes) == cudaSuccess &&
                    cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0;
    if (!ok) (void)cudaGetLastError();
    is = ok ? 1 : 2;
    known[dev].store(is, std::memory_order_release);
  }
  return is == 1;
}

int evict(const FaPagedEvictArgs* a, void* stream) {
  int rc = check_evict(a);
  if (rc != FA_OK) return rc;
  FaPagedCache c = a->cache;
  c.offsets = c.kv_lens;  // (there are no packed rows)
  const bool f8 = c.dtype == FA_DTYPE_FP8_E4M3;
  if (c.seqs == 0) return FA_OK;
  rc = check_cache(c, f8 ? FA_DTYPE_BF16 : c.dtype, 0);
  if (rc != FA_OK) return rc;
  if (!a->weights || !a->new_lens || (a->keep > 0 && !a->kept) || (!a->in_place && a->to_cols > 0 && !a->to_table))
    return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a->weights) % 16 || reinterpret_cast<uintptr_t>(a->workspace) % 256)
    return FA_ERR_MISALIGNED;
  const EvictChoice choice = choose(a);
  if (!a->workspace || a->workspace_bytes < choice.bytes) return FA_ERR_INVALID_ARG;
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
  p.lanes_log2 = choice.lanes_log2;
  p.rows = choice.rows;
  for (int i = 0; i < 2; ++i) p.chunks[i] = choice.chunks[i];
  p.ticket = static_cast<uint32_t*>(a->workspace);
  p.flags = a->in_place && !choice.in_order ? p.ticket + 64 : nullptr;
  const int sms = sm_count_of_current();
  const int64_t items = c.seqs * c.heads_kv, capacity = c.table_cols * c.page_size;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);

  // A (sequence, head) gets more CTAs while all of them find a place and have 2048 keys each.
  int cluster = 1;
  while (cluster < kMostCluster && items * cluster * 2 <= 2 * sms && capacity > 2048 * cluster) cluster *= 2;
  if (cluster > 8 && !large_clusters()) cluster = 8;
  const int64_t share = ((capacity + cluster - 1) / cluster + 3) / 4 * 4 + 4;
  const bool many = share > 8192 || cluster > 8;
  const int cols = many ? 4 : 1, threads = many ? 1024 : 512;
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
  return launch_dependent(choice.in_order ? choice.lanes_log2 >= 2 ? paged_move_in_order_kernel<1>
                                                                   : paged_move_in_order_kernel<2>
                                          : paged_move_kernel,
                          dim3(static_cast<unsigned>(choice.blocks)), kMoveThreads, 0, s, p);
}

}  // namespace
}  // namespace fa

extern "C" {

int64_t fa_paged_evict_workspace_bytes(const FaPagedEvictArgs* a) {
  const int rc = fa::check_evict(a);
  return rc != FA_OK ? rc : fa::choose(a).bytes;
}

int fa_paged_evict_sm100(const FaPagedEvictArgs* args, void* stream) { return fa::evict(args, stream); }

}  // extern "C"
