// Division of a paged attention call among CTAs, shared by its kernels.
//
// An item is one (sequence, kv head, block of query rows); it has one step per tile of keys (and
// one if there is no key, so that its rows are written), behind `item_cost` empty steps that stand
// for what an item costs besides its tiles (fetching the queries, joining, writing).  All steps of a call, in the order
// sequence - kv head - row block - key tile, form one line that is cut into equal ranges, one per
// CTA: ragged lengths, few sequences and long contexts all load the SMs alike, and only the two
// items at a CTA's ends can be shared with a neighbour.  Lengths are device data, so each CTA
// derives its range itself from two sums over the sequences.
//
// A CTA that holds a whole item writes its output.  A shared item's parts go to the workspace,
// normalised, in fp32, with their base-2 logsumexp: slot 0 of a CTA is the item that began before
// its range, slot 1 the one that goes on behind it.  paged_combine_kernel then joins them:
//   lse = log2 sum_i 2^lse_i ,   O = sum_i 2^(lse_i - lse) O_i ,
// in the order of the key tiles, so the result does not depend on timing.  That launch costs 3 to 5 us
// even where little is to be joined, so calls of short sequences do without (`whole_items`).
#pragma once

#include <climits>

#include "fa_fwd_kernel.cuh"
#include "fa_paged_common.cuh"

namespace fa {

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// Programmatic dependent launch: a kernel of the paged calls is brought up while the one before it
// in the stream still runs, and waits here for its end (and its memory) before it reads anything.
__device__ __forceinline__ void wait_for_launch_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// From here on the next kernel may be brought up.
__device__ __forceinline__ void let_next_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// What a CTA notes about its slot 0 for the combine kernel.
struct PagedPart {
  int first_cta; // CTA that holds the item's first part, in its slot 1; negative: slot 0 is empty
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
  uint32_t group_inv;  // floor(2^32 / group) + 1: n / group = umulhi(n, .) for n * group < 2^32,
                       // group > 1
  int head_dim;
  int causal;
  float scale_log2;  // sm_scale * log2(e)
  int min_steps_log2;  // steps of a CTA's range, at least
  int item_cost;     // empty steps before an item's tiles
  int whole_items;   // a CTA takes the items that begin in its range, whole: nothing is shared
  int tile_live;     // rows of a tile that are used: a multiple of `group` in the tile kernel
  int tile_toks;     // tokens of a tile (tile kernel)
  int pair_from;     // steps from which a part of one tile is worked on by both sides, at least 2
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

// Work of the row kernel: blocks of ROWS rows, each over all key tiles of its sequence.
template <int ROWS, int KEYS>
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnParams& p, int b) {
  PagedSeq s;
  seq_rows(p.seqs, b, s.first, s.count);
  s.len = seq_len(p.seqs, b);
  const int rows = s.count * p.group;  // at most total * heads_q, which the host bounds
  s.blocks = (rows + ROWS - 1) / ROWS;
  s.tiles = max(1, (s.len + KEYS - 1) / KEYS);
  s.steps = static_cast<int64_t>(p.heads_kv) * s.blocks * (s.tiles + p.item_cost);
  return s;
}

// Quotient of non-negative numbers, by the short division where they allow it (the long one takes
// ~150 cycles, which a call of a few microseconds would see several times).
__device__ __forceinline__ int64_t quot(int64_t a, int b) {
  return (a >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b))
                        : a / b;
}

// A CTA's range of the line, and where it begins.
struct PagedRange {
  int64_t lo, hi;  // steps
  int64_t base;    // first step of sequence `seq`
  int64_t all;     // steps of the call
  int64_t share;   // steps of a CTA, one more for the first `rest`
  int rest;
  int ctas;        // CTAs with a range
  int seq;

  // CTA whose range holds a step
  __device__ __forceinline__ int cta_of(int64_t step) const {
    const int64_t more = rest * (share + 1);  // steps of the CTAs that take one more
    const int64_t at = step < more ? step : step - more;
    const int64_t each = step < more ? share + 1 : share;
    const int64_t n = (at | each) >> 31 ? at / each : quot(at, static_cast<int>(each));
    return static_cast<int>(step < more ? n : rest + n);
  }
};

// steps_of(b): steps of sequence b.  Every warp of the CTA finds the range by itself, a lane for
// each 32nd of the sequences: two sums with a block barrier between them took longer than reading
// the same few lines in every warp.
template <typename Steps>
__device__ __forceinline__ PagedRange paged_range(const PagedAttnParams& p, Steps steps_of) {
  const int lane = threadIdx.x & 31;
  const int seqs = p.seqs.seqs;
  const int each = (seqs + 31) / 32;
  const int b0 = min(lane * each, seqs), b1 = min(b0 + each, seqs);
  int64_t own = 0;
  for (int b = b0; b < b1; ++b) own += steps_of(b);
  int64_t upto = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += v;
  }
  PagedRange r{0, 0, 0, __shfl_sync(0xffffffffu, upto, 31), 1, 0, 0, 0};
  const int64_t most = (r.all + (1 << p.min_steps_log2) - 1) >> p.min_steps_log2;
  r.ctas = static_cast<int>(most < gridDim.x ? most : gridDim.x);
  const int c = static_cast<int>(blockIdx.x);
  if (c >= r.ctas) return r;
  // the first `rest` CTAs take a step more than the others
  r.share = quot(r.all, r.ctas);
  r.rest = static_cast<int>(r.all - r.share * r.ctas);
  r.lo = r.share * c + min(c, r.rest);
  r.hi = r.lo + r.share + (c < r.rest);
  // the one lane whose sequences hold step `lo`
  int64_t from = upto - own;
  const bool mine = from <= r.lo && r.lo < upto;
  int b = b0;
  if (mine && each > 1) {
    for (int64_t n; from + (n = steps_of(b)) <= r.lo; ++b) from += n;
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
  r.seq = __shfl_sync(0xffffffffu, b, src);
  r.base = __shfl_sync(0xffffffffu, from, src);
  return r;
}

// Walks the items of a CTA's range; every role of the kernel walks the same ones.
template <int ROWS, int KEYS>
struct PagedWalk {
  const PagedAttnParams& p;
  const PagedRange& range;
  int64_t pos;       // next step of the line
  int at;            // ... and of the item
  int b;
  PagedSeq s;
  // the current part
  int head, block;
  int tile0, tile1;  // key tiles [tile0, tile1) of the item
  int64_t item;      // the item's first step

  __device__ __forceinline__ PagedWalk(const PagedAttnParams& params, const PagedRange& r)
      : p(params), range(r), pos(r.lo), b(r.seq) {
    if (pos >= range.hi) return;
    s = paged_seq<ROWS, KEYS>(p, b);
    const int64_t in_seq = pos - r.base;
    const int64_t n = quot(in_seq, s.tiles + p.item_cost);
    at = static_cast<int>(in_seq - n * (s.tiles + p.item_cost));
    head = static_cast<int>(s.blocks == 1 ? n : quot(n, s.blocks));
    block = static_cast<int>(n - static_cast<int64_t>(head) * s.blocks);
    if (p.whole_items && at > 0) {
      pos += s.tiles + p.item_cost - at;
      at = s.tiles + p.item_cost;
    }
  }
  __device__ __forceinline__ bool next() {
    do {
      if (pos >= range.hi) return false;
      if (at == s.tiles + p.item_cost) {
        at = 0;
        if (++block == s.blocks) {
          block = 0;
          if (++head == p.heads_kv) {
            head = 0;
            do s = paged_seq<ROWS, KEYS>(p, ++b);
            while (s.blocks == 0);
          }
        }
      }
      const int end = s.tiles + p.item_cost;
      const int64_t left = range.hi - pos;
      const int to = static_cast<int>(!p.whole_items && left < end - at ? at + left : end);
      tile0 = max(0, at - p.item_cost);
      tile1 = max(0, to - p.item_cost);
      item = pos - at;
      pos += to - at;
      at = to;
    } while (tile0 == tile1);  // empty steps only
    return true;
  }
  __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == s.tiles; }
  __device__ __forceinline__ int slot() const { return tile0 == 0 ? 1 : 0; }
  // What the combine kernel has to know of the current part (slot 0).
  __device__ __forceinline__ PagedPart note() const {
    return PagedPart{range.cta_of(item + p.item_cost),
                     range.cta_of(item + p.item_cost + s.tiles - 1), s.first, s.count, head, block};
  }
};

// Work of the tile kernel: blocks of TILES tiles of `tile_toks` tokens with all their heads, each
// over the key tiles up to its last token's position (causal) or the sequence's end.
template <int TILES, int KEYS>
struct PagedTiles {
  int first, count, len;
  int blocks;
  int64_t per_head;  // steps of one kv head

  // Key tiles that the tokens before `tok_end` attend to; 1 if there is none.
  __device__ __forceinline__ int tiles(const PagedAttnParams& p, int tok_end) const {
    const int end = p.causal ? min(len, len - count + min(tok_end, count)) : len;
    return max(1, (end + KEYS - 1) / KEYS);
  }
  __device__ __forceinline__ int block_tiles(const PagedAttnParams& p, int block) const {
    return tiles(p, (block + 1) * TILES * p.tile_toks);
  }
  PagedTiles() = default;
  __device__ __forceinline__ PagedTiles(const PagedAttnParams& p, int b) {
    seq_rows(p.seqs, b, first, count);
    len = seq_len(p.seqs, b);
    blocks = (count + TILES * p.tile_toks - 1) / (TILES * p.tile_toks);
    per_head = static_cast<int64_t>(blocks) * p.item_cost;
    if (!p.causal) {
      per_head += static_cast<int64_t>(blocks) * block_tiles(p, 0);
    } else {
      for (int m = 0; m < blocks; ++m) per_head += block_tiles(p, m);
    }
  }
  __device__ __forceinline__ int64_t steps(const PagedAttnParams& p) const {
    return per_head * p.heads_kv;
  }
};

// (plain data: it lives in shared memory)
template <int TILES, int KEYS>
struct PagedTileWalk {
  int64_t pos;       // next step of the line
  int at;            // ... and of the item
  int b;
  PagedTiles<TILES, KEYS> s;
  // the current part
  int head, block;
  int n;             // key tiles of the item
  int tile0, tile1;  // those of the part
  int64_t item;      // the item's first step

  PagedTileWalk() = default;
  __device__ __forceinline__ PagedTileWalk(const PagedAttnParams& p, const PagedRange& r)
      : pos(r.lo), b(r.seq) {
    if (pos >= r.hi) return;
    s = PagedTiles<TILES, KEYS>(p, b);
    int64_t in_seq = pos - r.base;
    head = static_cast<int>(s.per_head >> 31 ? in_seq / s.per_head
                                             : quot(in_seq, static_cast<int>(s.per_head)));
    in_seq -= head * s.per_head;
    block = 0;
    for (n = s.block_tiles(p, 0); in_seq >= n + p.item_cost; n = s.block_tiles(p, ++block))
      in_seq -= n + p.item_cost;
    at = static_cast<int>(in_seq);
    if (p.whole_items && at > 0) {
      pos += n + p.item_cost - at;
      at = n + p.item_cost;
    }
  }
  __device__ __forceinline__ bool next(const PagedAttnParams& p, int64_t hi) {
    do {
      if (pos >= hi) return false;
      if (at == n + p.item_cost) {
        at = 0;
        if (++block == s.blocks) {
          block = 0;
          if (++head == p.heads_kv) {
            head = 0;
            do s = PagedTiles<TILES, KEYS>(p, ++b);
            while (s.blocks == 0);
          }
        }
        n = s.block_tiles(p, block);
      }
      const int end = n + p.item_cost;
      const int64_t left = hi - pos;
      const int to = static_cast<int>(!p.whole_items && left < end - at ? at + left : end);
      tile0 = max(0, at - p.item_cost);
      tile1 = max(0, to - p.item_cost);
      item = pos - at;
      pos += to - at;
      at = to;
    } while (tile0 == tile1);  // empty steps only
    return true;
  }
  // First token of tile i of the block, and the steps of this part that the tile takes part in.
  __device__ __forceinline__ int tok0(const PagedAttnParams& p, int i) const {
    return (block * TILES + i) * p.tile_toks;
  }
  __device__ __forceinline__ int steps(const PagedAttnParams& p, int i) const {
    if (tok0(p, i) >= s.count) return 0;
    return min(max(s.tiles(p, tok0(p, i) + p.tile_toks) - tile0, 0), tile1 - tile0);
  }
  // Only the block's first tile has tokens: both sides of the CTA work on it, key tiles in turn.
  __device__ __forceinline__ bool paired(const PagedAttnParams& p) const {
    return TILES == 2 && tok0(p, 1) >= s.count && tile1 - tile0 >= p.pair_from;
  }
  // The part's last tile goes past the sequence's end.
  __device__ __forceinline__ bool tail() const { return tile1 * KEYS > s.len; }
  __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == n; }
  __device__ __forceinline__ int slot() const { return tile0 == 0 ? 1 : 0; }
  __device__ __forceinline__ PagedPart note(const PagedRange& r, int cost) const {
    return PagedPart{r.cta_of(item + cost), r.cta_of(item + cost + n - 1), s.first, s.count, head, block};
  }
};

// Several warps issue the copies of one stage.  When a wait of theirs gives up, they stop at the
// same stage, so that every phase that one of them has begun completes and can be drained: each
// comes here once, giving up or done, and those behind catch up with the farthest (which has seen
// the stages in between free).
template <int WARPS>
struct ProducersMeet {
  int* issued;   // shared, one word per warp
  uint32_t bar;  // named barrier
  int limit = INT_MAX;
  bool met = false;
  __device__ __forceinline__ void operator()(int warp, int count) {
    if (met) return;
    met = true;
    if ((threadIdx.x & 31) == 0) issued[warp] = count;
    named_barrier_sync(bar, WARPS * 32);
    limit = 0;
    for (int w = 0; w < WARPS; ++w) limit = max(limit, issued[w]);
  }
};

// Joins the parts of shared items.  An item has TILES tiles of TILE rows.  An item of n parts has
// n - 1 CTAs that continue it; blocks (c, y) belong to CTA c + 1 and take every (n - 1)-th row of
// its item, so that each CTA's blocks have about the same to read however often items are cut.
// WARPS warps to a row, which take every WARPS-th part each.
template <typename T, int TILE, int TILES, int WARPS, int ROWS>
__global__ void __launch_bounds__(WARPS * ROWS * 32)
    paged_combine_kernel(const PagedAttnParams p) {
  wait_for_launch_before();
  __shared__ float s_o[ROWS][WARPS][256];
  const int c = blockIdx.x + 1;
  const PagedPart part = p.parts[c];
  if (part.first_cta < 0) return;
  const int step = part.last_cta - part.first_cta;  // CTAs that share the rows
  const int n = step + 1;  // parts: slot 1 of first_cta, then slots 0 up to last_cta
  const int lane = threadIdx.x & 31;
  const int mine = threadIdx.x / (WARPS * 32);  // row of the block
  const int warp = (threadIdx.x >> 5) % WARPS;
  const int D = p.head_dim;
  for (int turn = blockIdx.y * ROWS; turn * step < TILE * TILES; turn += gridDim.y * ROWS) {
    const int row = (turn + mine) * step + (c - part.first_cta - 1);
    const int in_tile = row % TILE;
    const int at = (part.block * TILES + row / TILE) * p.tile_live + in_tile;
    const bool live = row < TILE * TILES && in_tile < p.tile_live && at < part.count * p.group;
    auto slot_row = [&](int i) -> int64_t {
      const int64_t slot = i == 0 ? static_cast<int64_t>(part.first_cta) * 2 + 1
                                  : static_cast<int64_t>(part.first_cta + i) * 2;
      return slot * (TILE * TILES) + row;
    };
    float acc[8];  // columns 32 k + lane
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
    float top = -INFINITY, sum = 0.f;
    if (live) {
      for (int i = lane; i < n; i += 32) top = fmaxf(top, p.part_lse[slot_row(i)]);
#pragma unroll
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float base = top == -INFINITY ? 0.f : top;  // no part has a key: all weights are 0
      for (int i = lane; i < n; i += 32) sum += exp2f(p.part_lse[slot_row(i)] - base);
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 4
      for (int i = warp; i < n; i += WARPS) {
        const int64_t r = slot_row(i);
        const float w = exp2f(p.part_lse[r] - base) * inv;
        if (w == 0.f) continue;  // a part without keys for the row may have left no values
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int d = k * 32 + lane;
          if (k * 32 < D && d < D) acc[k] += w * p.part_o[r * D + d];
        }
      }
    }
    const int64_t tok = part.first_row + at / p.group;
    const int64_t head = part.head_kv * p.group + at % p.group;
    T* out = static_cast<T*>(p.o) + tok * p.o_stride[0] + head * p.o_stride[1];
    if constexpr (WARPS > 1) {
      __syncthreads();  // the last row's sums have been read
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k * 32 + lane < D) s_o[mine][warp][k * 32 + lane] = acc[k];
      __syncthreads();
      if (live)
        for (int d = warp * 32 + lane; d < D; d += WARPS * 32) {
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) v += s_o[mine][w][d];
          out[d] = static_cast<T>(v);
        }
    } else if (live) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k * 32 + lane < D) out[k * 32 + lane] = static_cast<T>(acc[k]);
    }
    if (live && warp == 0 && lane == 0)
      p.lse[tok * p.heads_kv * p.group + head] = (top + log2f(sum)) * kLn2;
  }
}

}  // namespace fa
