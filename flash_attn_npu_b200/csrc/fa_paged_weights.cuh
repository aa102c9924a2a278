// The attention weight that each cached token received (fa_paged_weights_sm100 of
// include/fa_paged_sm100.h): per (sequence, kv head, key j), over the query rows i of the sequence that see
// the key and share the kv head,
//   w_j (+)= sum_i 2^(q_i k_j * scale * log2 e - l_i) ,   l_i = log2 e * (the attention call's logsumexp).
//
// The product is formed transposed, S^T [128 keys x rows] = K Q^T with tcgen05.mma: a thread of the
// epilogue owns a key (a TMEM lane) and adds along the rows, so there is no reduction between threads, no
// softmax state and nothing that one step has to wait for from the one before.  It also keeps everything
// apart that must not mix: what lies in the cache behind a sequence's end, or in rows of the query tile
// that are not the sequence's, stays in lanes and columns that nobody reads.
//
// An item is one (sequence, kv head, block of 256 keys), one key tile for each of two warpgroups; its steps
// are the query tiles (`tile_toks` tokens with all heads of the group) from the first one that a causal mask
// leaves.  K stays in shared memory for the item and Q streams through a ring; where a sequence has one
// query tile (decoding) Q stays and K streams, and every key is read once.  CTAs take equal ranges of the
// line of all steps (fa_paged_attn.cuh); an item that two or more CTAs share leaves its sums in the
// workspace, and paged_weights_join_kernel adds them up in the order of the steps, so the result does not
// depend on timing.
//
// Float8: the codes are exact in q's type and are converted as they are; the row's scale multiplies the
// thread's logits.
//
// Each key tile has two warpgroups, which take every other step (and TMEM buffer): the latency of a step is
// a few times its work.  What they add up is joined at the item's end.
//
// Warps (16-bit 20, or 24 where the sequences have one query tile; float8 28):
//   0-3, 4-7, 8-11, 12-15  epilogue: key tile 0 and 1 of even steps, key tile 0 and 1 of odd ones
//   16, 17    MMA issuers of key tile 0 and 1 (the first owns TMEM)
//   18        TMA producer of K (16 bits: of key tile 0; of 24: idle)
//   19        walks the line and tells the others the parts (a ring of descriptions: every warp walking
//             by itself took 1500 cycles an item); TMA producer of Q, and the logsumexps of its rows, and
//             (16 bits, of 20) of K's key tile 1
//   20-23     of 24: TMA producers of K, two for each key tile.  With one query tile an item is over as soon as its
//             keys are there, and walking while loading held them up: 64 single tokens took 148 us and then
//             117.  Prompts take 111 us with 20 warps and 123 with 24.
//   20-27     float8: convert the key tiles
// Measured: 64 single tokens over 500 to 8192 tokens (32 / 8 heads x 128, 16 bits) 119 us, 5.3 TB/s; 16 over 100 to
// 2000 in float8 23 us, the chain of an item; 5 prompts of 700 to 3500 tokens 112 us, 45 % of the
// exponential unit and 33 % of the tensor cores; 4 chunks of 300 to 1024 over 4096 to 16384 (16 / 4 heads x 64,
// float8) 166 us, 64 % of the exponential unit.
//
// What a ring holds is waited for and given back by all warps that read from it, in order, though not all
// look at each fill: a warp that passed over fills could take an older one for its own.
#pragma once

#include <type_traits>

#include "fa_paged_tile.cuh"

namespace fa {

struct PagedWeightsNote {
  int first_cta;  // CTA that holds the item's first part (in slot 1); negative: nothing to join
  int seq, head_kv, block;
};

struct PagedWeightsParams : PagedAttnParams {  // (o, lse, v: not used)
  const float* row_lse;       // [total, heads_q]
  float* weights;
  int64_t weights_stride[2];  // page, head
  int reset_new;              // places of the sequence's new tokens start from 0
  int chunks;                 // query tiles of a token: more than one where a group does not fit a tile
  int tile_heads;             // heads of a tile
  PagedWeightsNote* notes;    // [gridDim.x]
  float* parts;               // [gridDim.x][2][256]
};

constexpr int kWeightsBlock = 256;  // keys of an item

// ONE: of a 16-bit cache, a call whose sequences have one query tile (see `weights` in fa_paged_weights.cu).
template <int D, bool FP8, bool ONE = false>
struct WeightsGeo {
  static constexpr int QN = D <= 64 ? 128 : D == 128 ? (FP8 ? 64 : 128) : (FP8 ? 32 : 64);  // rows of a query tile
  static constexpr int ROW_BYTES = 2 * D;
  static constexpr int SWZ = ROW_BYTES >= 128 ? 128 : ROW_BYTES;
  static constexpr int NBLK = ROW_BYTES / SWZ;
  static constexpr int K_BLK = 128 * SWZ;
  static constexpr int K_TILE = 128 * ROW_BYTES;
  static constexpr int Q_BLK = QN * SWZ;
  static constexpr int Q_TILE = QN * ROW_BYTES;
  static constexpr int RAW = FP8 ? 128 * (D + 4) : 0;  // codes, scales
  static constexpr int K_SLOTS = D <= 64 ? (FP8 ? 3 : 4) : D == 128 ? 2 : 1;  // of each key tile of an item
  static constexpr int Q_SLOTS = D <= 64 && !FP8 ? 4 : 2;
  static constexpr int RAW_SLOTS = !FP8 ? 0 : D == 256 ? 1 : D == 128 ? 3 : 6;
  static constexpr int L_SLOTS = 2;  // logsumexps of query tiles, for steps of each parity
  static constexpr int I_SLOTS = 4;  // pages and scales of each key tile of an item
  static constexpr int P_SLOTS = 8;  // parts
  static constexpr int SHARED = 11 * 1024;
  static constexpr int TILES = 2 * K_SLOTS * K_TILE + Q_SLOTS * Q_TILE + RAW_SLOTS * RAW;
  // more than half of an SM's shared memory in any case: one CTA per SM, which takes all its TMEM
  static constexpr int SMEM = 1024 + TILES + SHARED > 120 * 1024 ? 1024 + TILES + SHARED : 120 * 1024;
  static constexpr int AUX = FP8 ? 8 : ONE ? 4 : 0;
  static constexpr int THREADS = (20 + AUX) * 32;
  // With AUX warps registers move to the epilogue (setmaxnreg).  Float8 has spilled at 72 a thread for all: 16 single
  // tokens took 25.5 us and take 23.5, chunks 182 and 165.  (88, with 72 for warps 16 to 19 and 40 for 20 to 27:
  // 23.1 and 169.)  16 bits: 117 us for 64 single tokens; 125 with 96, 56 and 40.
  static constexpr bool SPLIT = AUX > 0;
  static constexpr int REG_LAUNCH = FP8 ? 72 : 80, REG_EPILOGUE = FP8 ? 96 : 88, REG_ISSUE = FP8 ? 56 : 72,
                       REG_AUX = FP8 ? 32 : 56;
  static_assert(!SPLIT || 512 * REG_EPILOGUE + 128 * REG_ISSUE + AUX * 32 * REG_AUX <= THREADS * REG_LAUNCH,
                "register split");
  static constexpr int SHARE = ONE ? 2 : 1;  // producers of a key tile
  static constexpr uint32_t LAYOUT = SWZ == 128 ? 2u : SWZ == 64 ? 4u : 6u;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// One sequence's share of the line.
struct WeightsSeq {
  int first, count, len;
  int blocks;        // of 256 keys
  int full;          // ... that all query tiles may attend to, the first ones
  int qtiles;
  int64_t per_head;  // steps of one kv head

  WeightsSeq() = default;
  __device__ __forceinline__ WeightsSeq(const PagedWeightsParams& p, int b) {
    const int a = fresh(p.seqs.offsets + b), z = fresh(p.seqs.offsets + b + 1), n = fresh(p.seqs.kv_lens + b);
    first = min(max(a, 0), p.seqs.total);
    count = max(min(z, p.seqs.total) - first, 0);
    const int64_t cap = static_cast<int64_t>(p.seqs.table_cols) << p.seqs.page_log2;
    len = n < 0 ? 0 : static_cast<int>(n < cap ? n : cap);
    if (len != n || count != z - a) report(p.seqs.status, kStatusPageTable);
    blocks = count ? (len + kWeightsBlock - 1) / kWeightsBlock : 0;
    qtiles = (count + p.tile_toks - 1) / p.tile_toks * p.chunks;
    const int past = len - count;
    full = !p.causal ? blocks : past < 0 ? 0 : min(blocks, past / kWeightsBlock + 1);
    per_head = static_cast<int64_t>(full) * (qtiles + p.item_cost);
    for (int m = full; m < blocks; ++m) per_head += steps(p, m) + p.item_cost;
  }
  // First query tile that attends to a block, and how many do.
  __device__ __forceinline__ int first_q(const PagedWeightsParams& p, int block) const {
    return block < full ? 0 : (block * kWeightsBlock - (len - count)) / p.tile_toks * p.chunks;
  }
  __device__ __forceinline__ int steps(const PagedWeightsParams& p, int block) const {
    return qtiles - first_q(p, block);
  }
};

struct WeightsWalk {
  int64_t pos;  // next step of the line
  int at;       // ... and of the item
  int b;
  WeightsSeq s;
  // the current part
  int head, block;
  int n;        // query tiles of the item
  int q0;       // first one of them
  int t0, t1;   // those of the part: q0 + t0 .. q0 + t1
  int64_t item; // the item's first step

  WeightsWalk() = default;
  __device__ __forceinline__ WeightsWalk(const PagedWeightsParams& p, const PagedRange& r) : pos(r.lo), b(r.seq) {
    if (pos >= r.hi) return;
    s = WeightsSeq(p, b);
    int64_t in_seq = pos - r.base;
    head = static_cast<int>(s.per_head >> 31 ? in_seq / s.per_head : quot(in_seq, static_cast<int>(s.per_head)));
    in_seq -= head * s.per_head;
    const int each = s.qtiles + p.item_cost;
    block = static_cast<int>(min(quot(in_seq, each), static_cast<int64_t>(s.full)));
    in_seq -= static_cast<int64_t>(block) * each;
    for (n = s.steps(p, block); in_seq >= n + p.item_cost; n = s.steps(p, ++block)) in_seq -= n + p.item_cost;
    at = static_cast<int>(in_seq);
    if (p.whole_items && at > 0) {
      pos += n + p.item_cost - at;
      at = n + p.item_cost;
    }
  }
  __device__ __forceinline__ bool next(const PagedWeightsParams& p, int64_t hi) {
    do {
      if (pos >= hi) return false;
      if (at == n + p.item_cost) {
        at = 0;
        if (++block == s.blocks) {
          block = 0;
          if (++head == p.heads_kv) {
            head = 0;
            do s = WeightsSeq(p, ++b);
            while (s.blocks == 0);
          }
        }
        n = s.steps(p, block);
      }
      const int end = n + p.item_cost;
      const int64_t left = hi - pos;
      const int to = static_cast<int>(!p.whole_items && left < end - at ? at + left : end);
      t0 = max(0, at - p.item_cost);
      t1 = max(0, to - p.item_cost);
      item = pos - at;
      pos += to - at;
      at = to;
    } while (t0 == t1);
    q0 = s.first_q(p, block);
    return true;
  }
};

// A part as the warps see it: its sequence, what they need to know of it, and its steps.
struct alignas(16) WeightsPart {
  int tiles;   // key tiles with a key; 0: there is no further part
  int seq, head, block;
  int first, count, len;
  int qtile;   // first query tile
  int steps;
  int qtiles;  // of the sequence
  int slot;    // -1: a whole item, else that of the CTA's parts that its sums go to
  int note;    // this CTA holds an item's last part, and this one its first (-1: nothing to note)

  __device__ __forceinline__ int key0() const { return block * kWeightsBlock; }
  // A step's query tile: its first token, its first head of the group, and its rows.
  __device__ __forceinline__ int tok0(const PagedWeightsParams& p, int t) const {
    return (p.chunks == 1 ? qtile + t : (qtile + t) / p.chunks) * p.tile_toks;
  }
  __device__ __forceinline__ int head0(const PagedWeightsParams& p, int t) const {
    return p.chunks == 1 ? 0 : (qtile + t) % p.chunks * p.tile_heads;
  }
  __device__ __forceinline__ int rows(const PagedWeightsParams& p, int t) const {
    return min(count - tok0(p, t), p.tile_toks) * min(p.group - head0(p, t), p.tile_heads);
  }
};

template <typename G>
struct WeightsShared {
  uint64_t k_full[2][G::SHARE][G::K_SLOTS];  // from each producer
  uint64_t k_empty[2][G::K_SLOTS];
  uint64_t q_full[2][G::Q_SLOTS];  // copied; rows with l = -inf have been seen to
  uint64_t q_empty[G::Q_SLOTS];
  uint64_t l_full[2][G::L_SLOTS], l_empty[2][G::L_SLOTS];
  uint64_t i_full[2][G::I_SLOTS], i_empty[2][G::I_SLOTS];
  uint64_t p_full[G::P_SLOTS], p_empty[G::P_SLOTS];
  uint64_t raw_full[8], raw_empty[8];
  uint64_t s_full[2][2], s_empty[2][2];
  uint64_t sum_full[2][4], sum_empty[2][4];  // of a key tile, for each 32 of its keys
  uint64_t mma_done[2];
  WeightsPart parts[G::P_SLOTS];
  int page[2][G::I_SLOTS][16];       // of a key tile's boxes, -1: none
  int raw_page[8][16];
  float scale[2][G::I_SLOTS][128];   // float8: of a key tile's rows
  float sum[2][128];              // of the steps of the other warpgroup
  alignas(16) float neg_lse[2][G::L_SLOTS][G::QN];  // -l of a query tile's rows
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

// acc + 2^x of a pair on the FMA pipe: 2^(n - 1) 2^(f + 1) with n = round(x), f = x - n in [-1/2, 1/2], and twice the
// polynomial of degree 5 that minimises the relative error of 2^f there (the fit of exp2_poly_fit.py at degree 5:
// 2.3e-7, as ex2.approx; 5e-8 too large on average).  As 2^(n - 1) it is finite wherever 2^x is: up to 128.
// 0 below -125.5 (2^-127 has no bits in `scale`); NaN stays NaN.
__device__ __forceinline__ float2 add_exp2_poly(float2 x, float2 acc) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: the low bits of x + kRound are n
  constexpr float c0 = 2.000000238e+00f, c1 = 1.386293888e+00f, c2 = 4.804424047e-01f, c3 = 1.110142618e-01f,
                  c4 = 1.935108192e-02f, c5 = 2.655294258e-03f;
  auto both = [](float c) { return make_float2(c, c); };
  auto clamp = [](float v) {
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;\n\tmin.NaN.f32 %0, %0, 0f43000000;" : "+f"(v));  // -126, 128
    return v;
  };
  x = make_float2(clamp(x.x), clamp(x.y));
  const float2 t = fadd2(x, both(kRound));
  const float2 f = ffma2(fadd2(t, both(-kRound)), both(-1.f), x);
  float2 q = ffma2(both(c5), f, both(c4));
  q = ffma2(q, f, both(c3));
  q = ffma2(q, f, both(c2));
  q = ffma2(q, f, both(c1));
  q = ffma2(q, f, both(c0));
  const float2 scale = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f000000),
                                   __int_as_float((__float_as_int(t.y) << 23) + 0x3f000000));
  return ffma2(q, scale, acc);
}

template <typename T, int D, bool FP8, bool ONE>
__global__ void __launch_bounds__(WeightsGeo<D, FP8, ONE>::THREADS, 1)
    paged_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ PagedWeightsParams p) {
  using G = WeightsGeo<D, FP8, ONE>;
  using Sh = WeightsShared<G>;
  static_assert(sizeof(Sh) <= G::SHARED, "barrier block");
  constexpr int QN = G::QN, K_SLOTS = G::K_SLOTS, Q_SLOTS = G::Q_SLOTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* k_smem = smem;  // [2][K_SLOTS]
  uint8_t* q_smem = k_smem + 2 * K_SLOTS * G::K_TILE;
  uint8_t* raw_smem = q_smem + Q_SLOTS * G::Q_TILE;
  Sh* sh = reinterpret_cast<Sh*>(raw_smem + G::RAW_SLOTS * G::RAW);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* const status = p.seqs.status;

  let_next_launch();
  if (threadIdx.x == 0) {
    auto init = [](uint64_t* bars, int n, uint32_t count) {
      for (int s = 0; s < n; ++s) mbar_init(smem_u32(bars + s), count);
    };
    init(sh->k_full[0][0], 2 * G::SHARE * K_SLOTS, FP8 ? G::AUX : 1);
    init(sh->k_empty[0], 2 * K_SLOTS, 1);
    init(sh->q_full[0], 2 * Q_SLOTS, 1);
    init(sh->q_empty, Q_SLOTS, 2);  // the issuers
    init(sh->l_full[0], 2 * G::L_SLOTS, 1);
    init(sh->l_empty[0], 2 * G::L_SLOTS, 8);  // the epilogue of that parity
    init(sh->i_full[0], 2 * G::I_SLOTS, FP8 ? G::AUX : G::SHARE);
    init(sh->i_empty[0], 2 * G::I_SLOTS, 8);  // the two warpgroups of the tile
    init(sh->p_full, G::P_SLOTS, 1);
    init(sh->p_empty, G::P_SLOTS, (ONE ? 18 : 19) + G::AUX);  // all other warps that work
    init(sh->raw_full, 8, 1);
    init(sh->raw_empty, 8, G::AUX);
    init(sh->s_full[0], 4, 1);
    init(sh->s_empty[0], 4, 4);
    init(sh->sum_full[0], 8, 1);
    init(sh->sum_empty[0], 8, 1);
    init(sh->mma_done, 2, 1);
    sh->abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 16) {
    tmem_alloc(smem_u32(&sh->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  wait_for_launch_before();

  auto wait = [&](uint64_t& bar, uint32_t parity) {
    const bool ok = wait_bar_flag(&sh->abort_flag, smem_u32(&bar), parity, status);
    return static_cast<bool>(__all_sync(0xffffffffu, ok));
  };
  // The next part, in the order of the line; false: there is none, or a wait gave up.
  WeightsPart w;
  int pslot = 0;
  uint32_t pph = 0;
  auto next_part = [&]() -> bool {
    if (!wait(sh->p_full[pslot], pph)) return false;
    w = sh->parts[pslot];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh->p_empty[pslot]));
    if (++pslot == G::P_SLOTS) {
      pslot = 0;
      pph ^= 1u;
    }
    return w.tiles > 0;
  };
  // The query tile in use; a lone one stays from item to item of the same sequence and head.
  int q_seq = -1, q_head = -1;
  auto same_q = [&]() { return w.qtiles == 1 && q_seq == w.seq && q_head == w.head; };
  auto now_q = [&]() {
    q_seq = w.seq;
    q_head = w.head;
  };

  // Producer of key tiles: of both of an item, of one of them, or of every other page of one.
  // The copies of a tile, a lane each (two where the smallest pages have long rows).
  constexpr int COPIES = FP8 ? 2 : G::NBLK;  // of one page
  constexpr int SHARE = G::SHARE;
  constexpr int OPS = (16 / SHARE * COPIES + 31) / 32;
  struct Keys {
    int slot = 0, islot = 0;
    uint32_t ph = 0, iph = 0;
    int issued = 0;
    int ahead_seq = -1, ahead_block = -1;  // the item whose pages were fetched ahead
  };
  const int size = 1 << p.seqs.page_log2;
  const int box = min(size, 128);
  const int boxes = 128 / box;
  // (float8: `k` of the ring of raw tiles, which both key tiles share)
  auto load_keys = [&](int i, int half, Keys& k, int (&ahead)[OPS]) -> bool {
    const int key0 = w.key0() + i * 128;
    auto fetch = [&](int u, int first) {
      const int my_box = (lane + 32 * u) / COPIES * SHARE + half;
      const int pos = first + my_box * box;
      return my_box < boxes && pos < w.len ? page_entry(p.seqs, w.seq, pos) : -1;
    };
    const bool known = k.ahead_seq == w.seq && k.ahead_block == w.block;
    // the next block of the sequence, or the first one, of the next head
    const int next = w.key0() + kWeightsBlock < w.len ? w.block + 1 : 0;
    int entry[OPS];
#pragma unroll
    for (int u = 0; u < OPS; ++u) {
      entry[u] = known ? ahead[u] : fetch(u, key0);
      ahead[u] = fetch(u, next * kWeightsBlock + i * 128);
    }
    bool ok = FP8 ? wait(sh->raw_empty[k.slot], k.ph ^ 1u) : wait(sh->k_empty[i][k.slot], k.ph ^ 1u);
    if (!FP8 && ok) ok = wait(sh->i_empty[i][k.islot], k.iph ^ 1u);
    if (!ok) return false;
    const uint32_t bar = smem_u32(FP8 ? &sh->raw_full[k.slot] : &sh->k_full[i][half][k.slot]);
    const uint32_t dst = smem_u32(FP8 ? raw_smem + k.slot * G::RAW : k_smem + (i * K_SLOTS + k.slot) * G::K_TILE);
    int page[OPS];
#pragma unroll
    for (int u = 0; u < OPS; ++u) {
      const int my_box = (lane + 32 * u) / COPIES * SHARE + half, part = (lane + 32 * u) % COPIES;
      const bool in = my_box < boxes && key0 + my_box * box < w.len;
      page[u] = in ? checked_page(p.seqs, entry[u]) : -1;
      // (what is no page is copied from another one, and gets no weight)
      if (my_box < boxes && part == 0)
        (FP8 ? sh->raw_page[k.slot] : sh->page[i][k.islot])[my_box] = in && page[u] == entry[u] ? page[u] : -1;
    }
    __syncwarp();
    if (lane == 0) {  // (behind the page numbers, which those read who see the barrier complete)
      const int live = min(boxes, (w.len - key0 + box - 1) / box);  // with a key
      mbar_arrive_expect_tx(bar, (live - half + SHARE - 1) / SHARE * box * (FP8 ? D + 4 : G::ROW_BYTES));
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < OPS; ++u) {
      const int my_box = (lane + 32 * u) / COPIES * SHARE + half, part = (lane + 32 * u) % COPIES;
      const int row = (key0 + my_box * box) & (size - 1);
      if (page[u] < 0) continue;
      if constexpr (FP8) {
        if (part == 0) tma_load_4d(dst + my_box * box * D, &tmK, bar, 0, row, w.head, page[u]);
        else
          bulk_load_tile(dst + 128 * D + my_box * box * 4,
                         p.k_scale + page[u] * p.k_scale_stride[0] + w.head * p.k_scale_stride[1] + row, box * 4, bar);
      } else {
        tma_load_4d(dst + part * G::K_BLK + my_box * box * G::SWZ, &tmK, bar, part * (G::SWZ / 2), row, w.head, page[u]);
      }
    }
    __syncwarp();
    ++k.issued;
    if (++k.slot == (FP8 ? G::RAW_SLOTS : K_SLOTS)) {
      k.slot = 0;
      k.ph ^= 1u;
    }
    if constexpr (!FP8) {
      if (lane == 0) mbar_arrive(smem_u32(&sh->i_full[i][k.islot]));
      if (++k.islot == G::I_SLOTS) {
        k.islot = 0;
        k.iph ^= 1u;
      }
    }
    return true;
  };
  auto fetched = [&](Keys& k) {
    k.ahead_seq = w.seq;
    k.ahead_block = w.key0() + kWeightsBlock < w.len ? w.block + 1 : 0;
  };
  // The copies issued last land before shared memory goes away.
  auto drain_keys = [&](int i, int half, const Keys& k) {
    constexpr int RING = FP8 ? G::RAW_SLOTS : K_SLOTS;
    for (int u = 0; u < min(k.issued, RING); ++u) {
      const int x = k.issued - 1 - u;
      drain_bar(smem_u32(FP8 ? &sh->raw_full[x % RING] : &sh->k_full[i][half][x % RING]),
                static_cast<uint32_t>((x / RING) & 1));
    }
  };

  if constexpr (G::SPLIT) {
    if (warp >= 16 && warp < 20) setmaxnreg_dec<G::REG_ISSUE>();
  }
  if (warp == 18) {
    // ------------------------------------------------------------------ producer of K
    if constexpr (!ONE) {
      Keys k;
      int ahead[2][OPS];
      bool ok = true;
      while (ok && next_part()) {
#pragma unroll
        for (int i = 0; i < (FP8 ? 2 : 1); ++i)
          if (i < w.tiles && ok) ok = load_keys(i, 0, k, ahead[i]);
        if (FP8 && w.tiles == 1) k.ahead_block = -1;  // (those of the second tile have not been fetched)
        else fetched(k);
      }
      drain_keys(0, 0, k);
    }
  } else if (warp == 19) {
    // ------------------------------------------------------------------ the line, and Q
    if (lane == 0) p.notes[blockIdx.x].first_cta = -1;
    const PagedRange range =
        paged_range(p, [&](int b) { const WeightsSeq s(p, b); return s.per_head * p.heads_kv; });
    WeightsWalk walk(p, range);
    bool more = true, ok = true;
    // Tells the others the next part; it is told one part before its query tiles are loaded, so that its
    // keys are on their way while the part before is worked on.
    auto tell = [&](WeightsPart& x) {
      more = walk.next(p, range.hi);
      x = WeightsPart{};
      if (more) {
        x.tiles = walk.block * kWeightsBlock + 128 < walk.s.len ? 2 : 1;
        x.seq = walk.b;
        x.head = walk.head;
        x.block = walk.block;
        x.first = walk.s.first;
        x.count = walk.s.count;
        x.len = walk.s.len;
        x.qtile = walk.q0 + walk.t0;
        x.steps = walk.t1 - walk.t0;
        x.qtiles = walk.s.qtiles;
        x.slot = walk.t0 == 0 ? walk.t1 == walk.n ? -1 : 1 : 0;
        x.note = x.slot == 0 && walk.t1 == walk.n ? range.cta_of(walk.item + p.item_cost) : -1;
      }
      ok = wait(sh->p_empty[pslot], pph ^ 1u);
      if (!ok) return;
      if (lane == 0) {
        sh->parts[pslot] = x;
        mbar_arrive(smem_u32(&sh->p_full[pslot]));
      }
      if (++pslot == G::P_SLOTS) {
        pslot = 0;
        pph ^= 1u;
      }
    };
    int slot = 0, issued = 0, step = 0;  // (step: parity of the next one)
    int lslot[2] = {0, 0};
    uint32_t ph = 0, lph[2] = {0, 0};
    Keys k;
    int ahead[OPS];
    WeightsPart coming;
    tell(coming);
    while (ok && coming.tiles > 0) {
      w = coming;
      tell(coming);
      if (!FP8 && !ONE && w.tiles == 2) {
        if (ok) ok = load_keys(1, 0, k, ahead);
        fetched(k);
      }
      for (int t = 0; t < w.steps && ok; ++t, step ^= 1) {
        if (same_q()) continue;
        now_q();
        const int tok0 = w.tok0(p, t), head0 = w.head0(p, t), rows = w.rows(p, t);
        const float* const from = p.row_lse + static_cast<int64_t>(w.first + tok0) * (p.heads_kv * p.group) +
                                  w.head * p.group + head0;
        float l[QN / 32];
#pragma unroll
        for (int u = 0; u < QN / 32; ++u) {
          const int c = min(u * 32 + lane, rows - 1);  // (tile_heads = group unless tiles have one token)
          const int tok = p.chunks > 1 ? 0 : p.group == 1 ? c : static_cast<int>(__umulhi(c, p.group_inv));
          l[u] = fresh(from + static_cast<int64_t>(tok) * (p.heads_kv * p.group) + (c - tok * p.group));
        }
        ok = wait(sh->q_empty[slot], ph ^ 1u);
        if (!ok) break;
        if (lane == 0) {
          const uint32_t bar = smem_u32(&sh->q_full[0][slot]);
          mbar_arrive_expect_tx(bar, p.tile_toks * p.tile_heads * G::ROW_BYTES);
#pragma unroll
          for (int c = 0; c < G::NBLK; ++c)
            tma_load_3d(smem_u32(q_smem + slot * G::Q_TILE + c * G::Q_BLK), &tmQ, bar, c * (G::SWZ / 2),
                        w.head * p.group + head0, w.first + tok0);
        }
        // for steps of this parity, or for both where the tile stays
#pragma unroll
        for (int par = 0; par < 2; ++par) {
          if ((w.qtiles != 1 && par != step) || !ok) continue;
          ok = wait(sh->l_empty[par][lslot[par]], lph[par] ^ 1u);
          if (!ok) continue;
#pragma unroll
          for (int u = 0; u < QN / 32; ++u) {
            const bool none = u * 32 + lane >= rows || l[u] == -INFINITY;
            sh->neg_lse[par][lslot[par]][u * 32 + lane] = none ? -INFINITY : -l[u] * kLog2e;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->l_full[par][lslot[par]]));
          if (++lslot[par] == G::L_SLOTS) {
            lslot[par] = 0;
            lph[par] ^= 1u;
          }
        }
        // A row without keys, or left out by the caller (l = -inf), gives nothing whatever it holds: it becomes zeros, as
        // a logit that is not finite would get past -l.  (Here, and not where the logits are: leaving columns out in
        // the epilogue cost 64 single tokens 4 % and chunks 2 %; this costs 1.5 % and 0.6 %.)
        bool none = false;
#pragma unroll
        for (int u = 0; u < QN / 32; ++u) none |= l[u] == -INFINITY;
        if (__any_sync(0xffffffffu, none) && ok) {
          ok = wait(sh->q_full[0][slot], ph);
          if (ok) {
#pragma unroll
            for (int u = 0; u < QN / 32; ++u) {
              if (l[u] != -INFINITY) continue;
              // (the swizzle stays inside a row's SWZ bytes)
              uint8_t* const row = q_smem + slot * G::Q_TILE + (u * 32 + lane) * G::SWZ;
#pragma unroll 1
              for (int at = 0; at < G::ROW_BYTES; at += 16)
                *reinterpret_cast<uint4*>(row + at / G::SWZ * G::Q_BLK + at % G::SWZ) = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(smem_u32(&sh->q_full[1][slot]));
        ++issued;
        if (++slot == Q_SLOTS) {
          slot = 0;
          ph ^= 1u;
        }
      }
    }
    for (int u = 0; u < min(issued, Q_SLOTS); ++u) {
      const int x = issued - 1 - u;
      drain_bar(smem_u32(&sh->q_full[0][x % Q_SLOTS]), static_cast<uint32_t>((x / Q_SLOTS) & 1));
    }
    if constexpr (!FP8 && !ONE) drain_keys(1, 0, k);
  } else if (warp == 16 || warp == 17) {
    // ------------------------------------------------------------------ MMA issuers
    constexpr uint32_t hi = ((8u * G::SWZ) >> 4) | (1u << 14) | (G::LAYOUT << 29);
    const int i = warp - 16;
    const uint32_t k_lo = (smem_u32(k_smem + i * K_SLOTS * G::K_TILE) >> 4) | (1u << 16);
    const uint32_t q_lo = (smem_u32(q_smem) >> 4) | (1u << 16);
    int kslot = 0, qslot = -1, buf = 0;  // (buf: of the step)
    uint32_t kph = 0, qph = 1;           // (qph: of the slot in use)
    uint32_t sph[2] = {0, 0};
    bool held = false;  // a lone query tile's slot is given back when the next one comes
    bool ok = true;
    while (ok && next_part()) {
      const bool mine = i < w.tiles;
      for (int t = 0; t < w.steps && ok; ++t) {
        if (!same_q()) {
          now_q();
          if (held && lane == 0) mma_commit(smem_u32(&sh->q_empty[qslot]));
          held = w.qtiles == 1;
          if (++qslot == Q_SLOTS) qslot = 0;
          if (qslot == 0) qph ^= 1u;
#pragma unroll 1
          for (int x = 0; x < 2 && ok; ++x) ok = wait(sh->q_full[x][qslot], qph);
        }
        if (mine) {
#pragma unroll
          for (int half = 0; half < SHARE; ++half)
            if (t == 0 && ok) ok = wait(sh->k_full[i][half][kslot], kph);
          if (ok) ok = wait(sh->s_empty[i][buf], sph[buf] ^ 1u);
          if (!ok) break;
          sph[buf] ^= 1u;
          const int n = min(QN, (w.rows(p, t) + 15) & ~15);
          const uint32_t idesc = make_idesc(Elt<T>::kFmt, false, 128, 0) + (static_cast<uint32_t>(n >> 3) << 17);
          const uint32_t a0 = k_lo + ((kslot * G::K_TILE) >> 4);
          const uint32_t b0 = q_lo + ((qslot * G::Q_TILE) >> 4);
          const uint32_t d = tmem + (i * 2 + buf) * QN;
          tc_fence_after();
          if (lane == 0) {
#pragma unroll
            for (int c = 0; c < G::NBLK; ++c)
#pragma unroll
              for (int k = 0; k < G::SWZ / 32; ++k)
                mma_f16_ss_lo(d, a0 + ((c * G::K_BLK + k * 32) >> 4), b0 + ((c * G::Q_BLK + k * 32) >> 4), hi, idesc,
                              (c | k) ? 1u : 0u);
            mma_commit(smem_u32(&sh->s_full[i][buf]));
            if (t + 1 == w.steps) mma_commit(smem_u32(&sh->k_empty[i][kslot]));
          }
        }
        if (ok && !held && lane == 0) mma_commit(smem_u32(&sh->q_empty[qslot]));
        __syncwarp();
        buf ^= 1;
      }
      if (mine && ++kslot == K_SLOTS) {
        kslot = 0;
        kph ^= 1u;
      }
    }
    if (lane == 0) mma_commit(smem_u32(&sh->mma_done[i]));
    __syncwarp();
    drain_bar(smem_u32(&sh->mma_done[i]), 0);
  } else if (warp >= 20) {
    if constexpr (FP8) {
      // ---------------------------------------------------------------- convert the key tiles
      setmaxnreg_dec<G::REG_AUX>();
      // (lanes and pieces as in the tile kernel)
      constexpr int PR = D / 16;
      constexpr int LP = PR < 4 ? PR : 4;
      constexpr int RW = 32 / LP;
      constexpr int NG = PR / LP;
      constexpr int AT_ONCE = G::AUX * RW < 128 ? G::AUX * RW : 128;
      constexpr int STEPS = 128 / AT_ONCE;
      const int row0 = (warp - 20) * RW + lane / LP;
      const int group0 = row0 & (NG - 1);
      const int tid = threadIdx.x - 20 * 32;
      int slot[2] = {0, 0}, islot[2] = {0, 0}, rslot = 0;
      uint32_t ph[2] = {0, 0}, iph[2] = {0, 0}, rph = 0;
      bool ok = true;
      while (ok && next_part()) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i >= w.tiles || !ok) continue;
          ok = wait(sh->raw_full[rslot], rph) && wait(sh->i_empty[i][islot[i]], iph[i] ^ 1u) &&
               wait(sh->k_empty[i][slot[i]], ph[i] ^ 1u);
          if (!ok) continue;
          const uint8_t* raw = raw_smem + rslot * G::RAW;
          uint8_t* dst = k_smem + (i * K_SLOTS + slot[i]) * G::K_TILE;
          if (tid < 128) sh->scale[i][islot[i]][tid] = reinterpret_cast<const float*>(raw + 128 * D)[tid];
          if (tid < 16) sh->page[i][islot[i]][tid] = sh->raw_page[rslot][tid];
          if (row0 < AT_ONCE) {
#pragma unroll 1
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
              for (int s = 0; s < NG; ++s) {
                const int row = row0 + k * AT_ONCE;
                const int c = (group0 ^ s) * LP + lane % LP;
                const uint4 code = *reinterpret_cast<const uint4*>(raw + row * D + c * 16);
                const uint32_t cw[4] = {code.x, code.y, code.z, code.w};
                uint32_t out[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                  const uint32_t h2 = e4m3x2_to_h2(static_cast<uint16_t>(cw[u >> 1] >> (16 * (u & 1))));
                  if constexpr (std::is_same_v<T, __half>) {
                    out[u] = h2;
                  } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
                    out[u] = pack2(f.x, f.y, static_cast<T*>(nullptr));
                  }
                }
                uint8_t* blk = dst + (c * 32 / G::SWZ) * G::K_BLK;
                const uint32_t at = row * G::SWZ + (c * 32) % G::SWZ;
                *reinterpret_cast<uint4*>(blk + swizzle<G::SWZ>(at)) = make_uint4(out[0], out[1], out[2], out[3]);
                *reinterpret_cast<uint4*>(blk + swizzle<G::SWZ>(at + 16)) = make_uint4(out[4], out[5], out[6], out[7]);
              }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(&sh->i_full[i][islot[i]]));
            mbar_arrive(smem_u32(&sh->k_full[i][0][slot[i]]));
            mbar_arrive(smem_u32(&sh->raw_empty[rslot]));
          }
          if (++islot[i] == G::I_SLOTS) { islot[i] = 0; iph[i] ^= 1u; }
          if (++slot[i] == K_SLOTS) { slot[i] = 0; ph[i] ^= 1u; }
          if (++rslot == G::RAW_SLOTS) { rslot = 0; rph ^= 1u; }
        }
      }
    }
    if constexpr (ONE) {
      // ---------------------------------------------------------------- producers of K
      setmaxnreg_dec<G::REG_AUX>();
      const int i = warp >> 1 & 1, half = warp & 1;
      Keys k;
      int ahead[OPS];
      bool ok = true;
      while (ok && next_part()) {
        if (i >= w.tiles) continue;
        ok = load_keys(i, half, k, ahead);
        fetched(k);
      }
      drain_keys(i, half, k);
    }
  } else {
    // -------------------------------------------------------------------- epilogue
    if constexpr (G::SPLIT) setmaxnreg_inc<G::REG_EPILOGUE>();
    const int i = warp >> 2 & 1;     // key tile
    const int buf = warp >> 3;       // steps of this parity, and their buffer
    const int part = warp & 3;       // 32 keys of the tile
    const int r = threadIdx.x & 127; // key of the tile
    const uint32_t tS = tmem + (static_cast<uint32_t>(part * 32) << 16) + (i * 2 + buf) * QN;
    const int box_log2 = min(p.seqs.page_log2, 7);
    int islot = 0, lslot = -1, step = 0;  // (step: parity of the next one)
    uint32_t iph = 0, lph = 1, sph = 0, sum_ph = 0;
    bool ok = true;
    while (ok && next_part()) {
      // the warpgroup of the last step writes what both have added up
      const bool last = ((step + w.steps - 1) & 1) == buf;
      const bool mine = i < w.tiles && (w.steps > 1 || last);
      const int pos = w.key0() + i * 128 + r;
      const int past = w.len - w.count;
      float old = 0.f, k2 = p.scale_log2;
      float* place = nullptr;
      if (i < w.tiles) {
        ok = wait(sh->i_full[i][islot], iph);
        if (!ok) break;
        if (mine) {
          const int page = sh->page[i][islot][r >> box_log2];
          if (FP8) k2 *= sh->scale[i][islot][r];
          if (last && w.slot < 0 && pos < w.len && page >= 0) {
            place = p.weights + page * p.weights_stride[0] + w.head * p.weights_stride[1] + (pos & (size - 1));
            if (!(p.reset_new && pos >= past)) old = fresh(place);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->i_empty[i][islot]));
        if (++islot == G::I_SLOTS) {
          islot = 0;
          iph ^= 1u;
        }
      }
      const float2 kk = make_float2(k2, k2);
      float2 acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = make_float2(0.f, 0.f);
      for (int t = 0; t < w.steps && ok; ++t, step ^= 1) {
        if (!same_q()) {
          now_q();
          if (w.qtiles == 1 || step == buf) {
            __syncwarp();  // (lanes leave the last columns at their own pace)
            if (lslot >= 0 && lane == 0) mbar_arrive(smem_u32(&sh->l_empty[buf][lslot]));
            if (++lslot == G::L_SLOTS) lslot = 0;
            if (lslot == 0) lph ^= 1u;
            ok = wait(sh->l_full[buf][lslot], lph);
          }
        }
        if (i >= w.tiles || step != buf || !ok) continue;
        ok = wait(sh->s_full[i][buf], sph);
        if (!ok) break;
        sph ^= 1u;
        tc_fence_after();
        const int live = w.rows(p, t);
        // columns before `from` are hidden from this key: of tokens that come before it
        const int ahead = pos - past - w.tok0(p, t);
        const int from = p.causal ? max(0, ahead) * p.group : 0;
        const int from_all = p.causal ? max(0, ahead - lane + 31) * p.group : 0;
        const int from_any = p.causal ? max(0, ahead - lane) * p.group & ~31 : 0;
        const float* neg = sh->neg_lse[buf][lslot];
#pragma unroll 1
        for (int c0 = from_any; c0 < live; c0 += 32) {
          float s[32];
          tmem_ld32(tS + c0, reinterpret_cast<uint32_t*>(s));
          tmem_wait_ld();
#pragma unroll
          for (int u = 0; u < 32; ++u) asm volatile("" : "+f"(s[u]));
          if (c0 + 32 >= live) {  // the last of the buffer is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->s_empty[i][buf]));
          }
          if (c0 >= from_all && c0 + 32 <= live) {
#pragma unroll
            for (int u = 0; u < 32; u += 4) {
              const float4 l = *reinterpret_cast<const float4*>(neg + c0 + u);
              const float2 x = ffma2(make_float2(s[u], s[u + 1]), kk, make_float2(l.x, l.y));
              const float2 y = ffma2(make_float2(s[u + 2], s[u + 3]), kk, make_float2(l.z, l.w));
              float2& a = acc[u / 4 & 3];
              float2& b = acc[(u / 4 & 3) ^ 1];
              a = fadd2(a, make_float2(ex2_approx(x.x), ex2_approx(x.y)));
              if (FP8 || u / 4 % 2 != 0) b = fadd2(b, make_float2(ex2_approx(y.x), ex2_approx(y.y)));
              else b = add_exp2_poly(y, b);
            }
          } else {
#pragma unroll
            for (int u = 0; u < 32; u += 4) {
              if (c0 + u >= live) break;
              const float4 l = *reinterpret_cast<const float4*>(neg + c0 + u);
              const float x[4] = {fmaf(s[u], k2, l.x), fmaf(s[u + 1], k2, l.y), fmaf(s[u + 2], k2, l.z),
                                  fmaf(s[u + 3], k2, l.w)};
#pragma unroll
              for (int v = 0; v < 4; ++v)
                if (c0 + u + v >= from && c0 + u + v < live) acc[v].x += ex2_approx(x[v]);
            }
          }
        }
        if (from_any >= live) {  // (nothing to read)
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->s_empty[i][buf]));
        }
      }
      if (!mine || !ok) continue;
      const float2 a = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
      float sum = a.x + a.y;
      if (w.steps > 1) {
        uint64_t& full = sh->sum_full[i][part];
        uint64_t& empty = sh->sum_empty[i][part];
        ok = last ? wait(full, sum_ph) : wait(empty, sum_ph ^ 1u);
        if (!ok) break;
        sum_ph ^= 1u;
        if (last) sum += sh->sum[i][r];
        else sh->sum[i][r] = sum;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(last ? &empty : &full));
        if (!last) continue;
      }
      if (w.slot < 0) {
        if (place) *place = old + sum;
      } else {
        p.parts[(static_cast<int64_t>(blockIdx.x) * 2 + w.slot) * kWeightsBlock + i * 128 + r] = sum;
        if (i == 0 && r == 0 && w.note >= 0)
          p.notes[blockIdx.x] = PagedWeightsNote{w.note, w.seq, w.head, w.block};
      }
    }
  }

  // ---- teardown: every thread arrives here exactly once
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds up the parts of items that CTAs share: a block for each CTA, which works where the CTA holds an
// item's last part.
static __global__ void __launch_bounds__(kWeightsBlock) paged_weights_join_kernel(
    const __grid_constant__ PagedWeightsParams p) {
  wait_for_launch_before();
  const int c = blockIdx.x + 1;
  const PagedWeightsNote note = p.notes[c];
  if (note.first_cta < 0 || note.first_cta >= c) return;
  int first, count;
  seq_rows(p.seqs, note.seq, first, count);
  const int len = seq_len(p.seqs, note.seq);
  const int pos = note.block * kWeightsBlock + threadIdx.x;
  if (pos >= len) return;
  float sum = p.parts[(2 * static_cast<int64_t>(note.first_cta) + 1) * kWeightsBlock + threadIdx.x];
  for (int i = note.first_cta + 1; i <= c; ++i)
    sum += p.parts[2 * static_cast<int64_t>(i) * kWeightsBlock + threadIdx.x];
  const int page = page_of(p.seqs, note.seq, pos);
  if (page < 0) return;  // (reported by the kernel before)
  float* place = p.weights + page * p.weights_stride[0] + note.head_kv * p.weights_stride[1] +
                 (pos & ((1 << p.seqs.page_log2) - 1));
  const float old = p.reset_new && pos >= len - count ? 0.f : *place;
  *place = old + sum;
}

}  // namespace fa
