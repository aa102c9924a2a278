// Division of a paged attention call among CTAs, shared by its kernels.
//
// An item is one (sequence, kv head, block of query rows); it has one step per tile of keys (and
// one if there is no key, so that its rows are written).  All steps of a call, in the order
// sequence - kv head - row block - key tile, form one line that is cut into equal ranges, one per
// CTA: ragged lengths, few sequences and long contexts all load the SMs alike, and only the two
// items at a CTA's ends can be shared with a neighbour.  Lengths are device data, so each CTA
// derives its range itself from two sums over the sequences.
//
// A CTA that holds a whole item writes its output.  A shared item's parts go to the workspace,
// normalised, in fp32, with their base-2 logsumexp: slot 0 of a CTA is the item that began before
// its range, slot 1 the one that goes on behind it.  paged_combine_kernel then joins them:
//   lse = log2 sum_i 2^lse_i ,   O = sum_i 2^(lse_i - lse) O_i ,
// in the order of the key tiles, so the result does not depend on timing.
#pragma once

#include <climits>

#include "fa_fwd_kernel.cuh"
#include "fa_paged_common.cuh"

namespace fa {

// What a CTA notes about its slot 0 for the combine kernel.
struct PagedPart {
  int first_cta; // CTA that holds the item's first part, in its slot 1; -1: slot 0 is empty
  int last_cta;  // CTA that holds its last part
  int first_row; // packed row of the sequence's first query
  int count;     // queries of the sequence
  int head_kv;
  int block;     // row block
};

struct PagedAttnParams {
  PagedSeqs seqs;
  const void* q;
  void* o;
  float* lse;
  int64_t q_stride[2];
  int64_t o_stride[2];
  const float* k_scale;
  const float* v_scale;
  int64_t k_scale_stride[2];
  int64_t v_scale_stride[2];
  int heads_kv;
  int group;         // query heads per kv head
  int head_dim;
  int causal;
  float scale_log2;  // sm_scale * log2(e)
  int min_steps;     // steps of a CTA's range, at least
  int rows_from;     // this launch takes the sequences with rows_from <= count * group <= rows_to
  int rows_to;
  PagedPart* parts;  // [gridDim.x]
  float* part_o;     // [gridDim.x][2][block rows][head_dim]
  float* part_lse;   // [gridDim.x][2][block rows]
};

// One sequence's share of the line.
struct PagedSeq {
  int first, count, len;
  int blocks;  // row blocks
  int tiles;   // key tiles
  int64_t steps;
};

template <int ROWS, int KEYS>
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnParams& p, int b) {
  PagedSeq s;
  seq_rows(p.seqs, b, s.first, s.count);
  s.len = seq_len(p.seqs, b);
  const int rows = s.count * p.group;  // at most total * heads_q, which the host bounds
  s.blocks = (rows + ROWS - 1) / ROWS;
  s.tiles = max(1, (s.len + KEYS - 1) / KEYS);
  if (rows < p.rows_from || rows > p.rows_to) s.blocks = 0;
  s.steps = static_cast<int64_t>(p.heads_kv) * s.blocks * s.tiles;
  return s;
}

// A CTA's range of the line, and where it begins.
struct PagedRange {
  int64_t lo, hi;  // steps
  int64_t base;    // first step of sequence `seq`
  int64_t all;     // steps of the call
  int ctas;        // CTAs with a range
  int seq;
};

// By all threads of the CTA; `scratch`: 40 words of shared memory.
template <int ROWS, int KEYS>
__device__ __forceinline__ PagedRange paged_range(const PagedAttnParams& p, int64_t* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int threads = blockDim.x, warps = threads >> 5;
  const int mine = threadIdx.x;
  const int64_t first = mine < p.seqs.seqs ? paged_seq<ROWS, KEYS>(p, mine).steps : 0;
  int64_t sum = first;
  for (int b = mine + threads; b < p.seqs.seqs; b += threads)
    sum += paged_seq<ROWS, KEYS>(p, b).steps;
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) scratch[warp] = sum;
  __syncthreads();
  int64_t all = 0;
  for (int w = 0; w < warps; ++w) all += scratch[w];
  __syncthreads();

  PagedRange r{0, 0, 0, all, 0, 0};
  int64_t ctas = (all + p.min_steps - 1) / p.min_steps;
  if (ctas > gridDim.x) ctas = gridDim.x;
  r.ctas = static_cast<int>(ctas);
  const int64_t c = blockIdx.x;
  if (c >= ctas) return r;
  r.lo = all * c / ctas;
  r.hi = all * (c + 1) / ctas;
  int64_t before = 0;
  for (int at = 0; at < p.seqs.seqs; at += threads) {
    const int b = at + mine;
    const int64_t own =
        at == 0 ? first : (b < p.seqs.seqs ? paged_seq<ROWS, KEYS>(p, b).steps : 0);
    int64_t upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 31) scratch[warp] = upto;
    __syncthreads();
    int64_t chunk = 0, skip = 0;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) skip += scratch[w];
      chunk += scratch[w];
    }
    const int64_t from = before + skip + upto - own;
    if (from <= r.lo && r.lo < from + own) {
      scratch[33] = b;
      scratch[34] = from;
    }
    __syncthreads();
    before += chunk;
    if (before > r.lo) break;
  }
  r.seq = static_cast<int>(scratch[33]);
  r.base = scratch[34];
  return r;
}

// Walks the items of a CTA's range; every role of the kernel walks the same ones.
template <int ROWS, int KEYS>
struct PagedWalk {
  const PagedAttnParams& p;
  int64_t pos, hi, base, all;
  int ctas;
  int b;
  PagedSeq s;
  // the current part
  int head, block;
  int tile0, tile1;  // key tiles [tile0, tile1) of the item
  int64_t item;      // its first step

  __device__ __forceinline__ PagedWalk(const PagedAttnParams& params, const PagedRange& r)
      : p(params), pos(r.lo), hi(r.hi), base(r.base), all(r.all), ctas(r.ctas), b(r.seq) {
    if (pos < hi) s = paged_seq<ROWS, KEYS>(p, b);
  }
  __device__ __forceinline__ bool next() {
    if (pos >= hi) return false;
    while (pos >= base + s.steps) {
      base += s.steps;
      s = paged_seq<ROWS, KEYS>(p, ++b);
    }
    const int64_t at = pos - base;
    const int64_t n = at / s.tiles;
    tile0 = static_cast<int>(at - n * s.tiles);
    const int64_t left = hi - pos;
    tile1 = static_cast<int>(left < s.tiles - tile0 ? tile0 + left : s.tiles);
    head = static_cast<int>(n / s.blocks);
    block = static_cast<int>(n - static_cast<int64_t>(head) * s.blocks);
    item = pos - tile0;
    pos += tile1 - tile0;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == s.tiles; }
  __device__ __forceinline__ int slot() const { return tile0 == 0 ? 1 : 0; }
  // CTA whose range holds a step
  __device__ __forceinline__ int cta_of(int64_t step) const {
    return static_cast<int>(((step + 1) * ctas - 1) / all);
  }
  // What the combine kernel has to know of the current part (slot 0).
  __device__ __forceinline__ PagedPart note() const {
    return PagedPart{cta_of(item), cta_of(item + s.tiles - 1), s.first, s.count, head, block};
  }
};

// Joins the parts of shared items.  Block (c, r): row r of the item that CTA c continues, if it
// is the item's second part.  WARPS warps take every WARPS-th part each.
template <typename T, int ROWS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
    paged_combine_kernel(const PagedAttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float s_o[WARPS][256];
  const int c = blockIdx.x + 1;
  const int row = blockIdx.y;
  const PagedPart part = p.parts[c];
  if (part.first_cta != c - 1) return;
  const int at = part.block * ROWS + row;
  if (at >= part.count * p.group) return;
  const int n = part.last_cta - c + 2;  // slot 1 of CTA c - 1, then slots 0 of c .. last_cta
  auto slot_row = [&](int i) -> int64_t {
    const int64_t slot = i == 0 ? static_cast<int64_t>(c - 1) * 2 + 1
                                : static_cast<int64_t>(c - 1 + i) * 2;
    return slot * ROWS + row;
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, p.part_lse[slot_row(i)]);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float base = top == -INFINITY ? 0.f : top;  // no part has a key: all weights are 0
  float sum = 0.f;
  for (int i = lane; i < n; i += 32) sum += exp2f(p.part_lse[slot_row(i)] - base);
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);

  // each lane owns up to 8 values of the row
  const int D = p.head_dim;
  float acc[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) acc[k] = 0.f;
#pragma unroll 4
  for (int i = warp; i < n; i += WARPS) {
    const int64_t r = slot_row(i);
    const float w = exp2f(p.part_lse[r] - base) * inv;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = k * 32 + lane;
      if (k * 32 < D && d < D) acc[k] += w * p.part_o[r * D + d];
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k * 32 + lane < D) s_o[warp][k * 32 + lane] = acc[k];
  __syncthreads();
  const int64_t tok = part.first_row + at / p.group;
  const int64_t head = part.head_kv * p.group + at % p.group;
  T* out = static_cast<T*>(p.o) + tok * p.o_stride[0] + head * p.o_stride[1];
  for (int d = threadIdx.x; d < D; d += WARPS * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += s_o[w][d];
    out[d] = static_cast<T>(v);
  }
  if (threadIdx.x == 0)
    p.lse[tok * p.heads_kv * p.group + head] = (top + log2f(sum)) * kLn2;
}

}  // namespace fa
