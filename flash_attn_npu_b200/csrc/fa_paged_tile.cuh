// Paged attention of many query rows per kv head (prompts, chunks): bound by the tensor cores and
// the exponentials.
//
// Where a block has rows for one tile only, both sides (softmax warps, issuers, S and O in TMEM) work
// on that tile, each on every other key tile, and join their (m, l, O) at the part's end: a single
// side is a chain of MMA, exponentials, MMA that leaves the units idle more than half the time
// (~2900 cycles a step of 128 keys, where two sides take ~3700 for twice the work).
//
// A query tile is 128 rows of TMEM: `tile_toks` tokens times the `group` query heads that share a
// kv head (as many whole tokens as fit), so that grouped heads fill the tensor cores and share
// every key and value.  A CTA works on TILES tiles (two up to head_dim 128, one at 256) over the
// same keys and walks its range of key tiles (fa_paged_attn.cuh).  Per tile and step of KEYS keys:
//   S = Q K^T -> p = 2^(S * scale * log2 e - m), row sums l -> O += P V
// with S, P (16 bits, over S) and O in TMEM, tcgen05.mma throughout.
//
// Warps (16, float8 20):
//   0-3, 4-7  softmax of tile 0, 1 (thread r owns row r), rescaling and output
//   next 4    16-bit cache: clean the sequence's end
//   next 8    float8 cache: dequantise the tiles
//   last 4    MMA issuer of tile 0 (owns TMEM), TMA producer, MMA issuer of tile 1, TMA producer;
//             the issuers take turns
//
// Pages: the producer's lanes look a tile's pages up and each copies one (rows of at most 128
// bytes per copy).  What lies behind a sequence's last key may be any bits.  Its logits are
// masked, but 0 * NaN in P V is NaN, so those rows of V are zeroed in shared memory before the MMA
// reads them, by the helper warps on the last tile.
//
// Float8: tiles land in a ring of their own; the helper warps write code * scale, rounded to q's
// type (exact for the powers of two that the cache's writer leaves), as operands in the layout that
// TMA would have left.  That costs 1 (fp16) to 2.5 (bf16) instructions a value once per key tile, for
// both query tiles; four warps took ~1600 cycles a tile (two tiles a step), longer than a step of
// the rest, so there are eight.
//
// Softmax: exponentiate first, against the row's base, and look at the row sum; only a row whose
// sum is large takes its maximum, and moves its base if that passed it by 2^8, rescaling O itself
// (O is complete up to the last step once S of this step is).  fp16 probabilities carry 2^7.
//
// Measured (head_dim 128, 4 query heads a kv head, all SMs busy on caches of their own): a key tile
// takes two sides 2.0 us (16-bit cache) or 2.5 (float8), one side's rows on both sides 1.35 or 1.75.
// Four chunks of 3400 tokens in all over 50,000 in the cache, 8 kv heads: 670 us in a short run, 730 to 775 under
// the power limit, 1005 to 870 TFLOP/s (ncu: tensor pipe 56 %, exponentials 56 %); the persistent dense kernel
// with as many pairs, in turn with it, 640 to 700 and 646 to 674.  Twelve sequences of 1 to 226 new tokens
// over 59,000 in a float8 cache, 4 kv heads: 103 us; tiles of few rows leave the units idle (tensor pipe
// 20 %).  148 blocks of 256 rows over one key tile each: 12.6 us, most of it start and output.
//
// Tried for float8 and slower: half tiles as raw stages, so that four operand stages fit, with K and V
// rings of their own (112 us against 106 on the mixed batch); 2 KB pieces dealt out to four warps
// (142 us).  A line weighted by the query tiles of a block made most mixed batches 2 to 19 % slower,
// since few rows cost a float8 step nearly as much as many.
//
// Every wait is bounded as in the dense kernels: a wait that gives up sets the status word and
// the CTA's abort flag, all roles fall through to the teardown, which drains copies and MMAs.
#pragma once

#include <type_traits>

#include "fa_paged_attn.cuh"

namespace fa {

template <int D, bool FP8>
struct TileGeo {
  static constexpr int TILES = D <= 128 ? 2 : 1;
  static constexpr int KEYS = D <= 128 ? 128 : 64;
  static constexpr int ROW_BYTES = 2 * D;
  static constexpr int SWZ = ROW_BYTES >= 128 ? 128 : ROW_BYTES;
  static constexpr int NBLK = ROW_BYTES / SWZ;       // swizzle spans of a row
  static constexpr int Q_BLK = 128 * SWZ;
  static constexpr int Q_TILE = 128 * ROW_BYTES;
  static constexpr int KV_BLK = KEYS * SWZ;
  static constexpr int KV_TILE = KEYS * ROW_BYTES;
  static constexpr int RAW = FP8 ? KEYS * (D + 4) : 0;  // codes, scales
  static constexpr int RAW_STAGES = FP8 ? 3 : 0;
  static constexpr int FIXED = 1024 + TILES * Q_TILE + RAW_STAGES * RAW + 5120;
  static constexpr int FIT = (227 * 1024 - FIXED) / KV_TILE;
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  // More than half of an SM's shared memory in any case: one CTA per SM, which takes all its TMEM.
  static constexpr int SMEM =
      FIXED + STAGES * KV_TILE > 120 * 1024 ? FIXED + STAGES * KV_TILE : 120 * 1024;
  static constexpr int TMEM_O = TILES * KEYS;
  // Warps: 0-7 softmax, AUX helpers (see above), then MMA, TMA, MMA, TMA; and the split of the
  // registers of the launch among the warpgroups.
  static constexpr int AUX = FP8 ? 8 : 4;
  static constexpr int MMA_WARP = 8 + AUX;
  static constexpr int THREADS = (12 + AUX) * 32;
  static constexpr int REG_LAUNCH = FP8 ? 96 : 128;
  static constexpr int REG_SOFTMAX = FP8 ? 168 : 192;
  static constexpr int REG_AUX = FP8 ? 48 : 64;
  static constexpr int REG_MISC = FP8 ? 48 : 64;
  static_assert(256 * REG_SOFTMAX + AUX * 32 * REG_AUX + 128 * REG_MISC <= THREADS * REG_LAUNCH,
                "register split");
  static constexpr uint32_t LAYOUT = SWZ == 128 ? 2u : SWZ == 64 ? 4u : 6u;
  static constexpr float P_OFFSET = 7.f;  // of fp16 probabilities: at most 2^(7 + 8) < 65504
  static_assert(STAGES >= 3, "K and V of a step, and one to come");
  static_assert(TMEM_O + TILES * D <= 512, "TMEM");
};

template <int STAGES, typename Walk>
struct TileShared {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[STAGES], kv_empty[STAGES];
  uint64_t v_go[STAGES];     // this slot's V goes past a sequence's end (16-bit caches) ...
  uint64_t v_clean[STAGES];  // ... and what lies there has been zeroed
  uint64_t raw_full[4], raw_empty[4];
  uint64_t s_full[2], p_ready[2], o_full[2], o_empty[2];
  uint64_t mma_done;
  float2 pair[2][128];  // (m, l) of the two sides' rows
  int issued[2];
  PagedRange range;
  Walk first_walk;  // at the CTA's first part, if there is one
  int first_more;
  Walk walks[20];  // one per warp: kept out of the registers of the roles' loops
  int more[20];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void bulk_load_tile(uint32_t dst, const void* src, uint32_t bytes,
                                               uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void st_global_v8(void* to, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <typename T, int D, bool FP8>
__global__ void __launch_bounds__(TileGeo<D, FP8>::THREADS, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tmQ,
                      const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedAttnParams p) {
  using G = TileGeo<D, FP8>;
  using Walk = PagedTileWalk<G::TILES, G::KEYS>;
  using Sh = TileShared<G::STAGES, Walk>;
  static_assert(sizeof(Sh) <= 5120, "barrier block");
  constexpr int TILES = G::TILES, KEYS = G::KEYS, STAGES = G::STAGES;
  constexpr bool kHalf = std::is_same_v<T, __half>;
  constexpr float kPOffset = kHalf ? G::P_OFFSET : 0.f;
  constexpr uint32_t IDESC_S = make_idesc(Elt<T>::kFmt, false, 128, KEYS);
  constexpr uint32_t IDESC_O = make_idesc(Elt<T>::kFmt, true, 128, D);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* q_smem = smem;
  uint8_t* kv_smem = q_smem + TILES * G::Q_TILE;
  uint8_t* raw_smem = kv_smem + STAGES * G::KV_TILE;
  Sh* sh = reinterpret_cast<Sh*>(raw_smem + G::RAW_STAGES * G::RAW);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int* const status = p.seqs.status;

  let_next_launch();
  if (threadIdx.x == 32) {
    prefetch_map(&tmQ);
    prefetch_map(&tmK);
    prefetch_map(&tmV);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&sh->kv_full[s]), FP8 ? G::AUX : 2);  // converting warps, or the producers
      mbar_init(smem_u32(&sh->kv_empty[s]), TILES);       // one commit per issuer
      mbar_init(smem_u32(&sh->v_go[s]), 1);
      mbar_init(smem_u32(&sh->v_clean[s]), 4);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(smem_u32(&sh->raw_full[s]), 2);
      mbar_init(smem_u32(&sh->raw_empty[s]), G::AUX);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh->q_full[i]), 1);
      mbar_init(smem_u32(&sh->q_empty[i]), 1);
      mbar_init(smem_u32(&sh->s_full[i]), 1);
      mbar_init(smem_u32(&sh->p_ready[i]), 4);
      mbar_init(smem_u32(&sh->o_full[i]), 1);
      mbar_init(smem_u32(&sh->o_empty[i]), 4);
    }
    mbar_init(smem_u32(&sh->mma_done), TILES);
    sh->abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == G::MMA_WARP) {
    tmem_alloc(smem_u32(&sh->tmem_base), 512);
    tmem_relinquish();
  }
  // Rows of the query tiles that no token fills are never written by a copy: they are zero.
  if (p.tile_live < 128) {
    for (int x = threadIdx.x * 16; x < TILES * G::Q_TILE; x += G::THREADS * 16)
      if ((x % G::Q_BLK) / G::SWZ >= p.tile_live)
        *reinterpret_cast<uint4*>(q_smem + x) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  wait_for_launch_before();
  if (threadIdx.x == 0) p.parts[blockIdx.x].first_cta = -2;
  if (warp == 0) {
    const PagedRange r =
        paged_range(p, [&](int b) { return PagedTiles<TILES, KEYS>(p, b).steps(p); });
    if (lane == 0) {
      sh->range = r;
      Walk x(p, r);
      sh->first_more = x.next(p, r.hi);
      sh->first_walk = x;
    }
  }
  __syncthreads();
  const PagedRange& range = sh->range;

  auto wait1 = [&](uint64_t& bar, uint32_t parity) {
    return wait_bar_flag(&sh->abort_flag, smem_u32(&bar), parity, status);
  };
  auto wait = [&](uint64_t& bar, uint32_t parity) {
    return static_cast<bool>(__all_sync(0xffffffffu, wait1(bar, parity)));
  };
  Walk& w = sh->walks[warp];
  bool begun = false;
  auto next_part = [&]() -> bool {
    __syncwarp();  // the warp is done with the last part
    if (lane == 0) {
      Walk x = begun ? w : sh->first_walk;
      sh->more[warp] = begun ? x.next(p, range.hi) : sh->first_more;
      w = x;
    }
    begun = true;
    __syncwarp();
    return sh->more[warp] != 0;
  };

  if (warp >= G::MMA_WARP) {
    setmaxnreg_dec<G::REG_MISC>();
    if (warp == G::MMA_WARP + 1 || warp == G::MMA_WARP + 3) {
      // ---------------------------------------------------------------- TMA producers
      // The copies of a tile, a lane each, spread over both warps (see the row kernel).
      const int pw = warp == G::MMA_WARP + 3;
      const int op = lane * 2 + pw;
      constexpr int COPIES = FP8 ? 2 : G::NBLK;  // of one page of K or V
      const int size = 1 << p.seqs.page_log2;
      const int box = min(size, KEYS);
      const int boxes = KEYS / box;
      const int my_box = op / COPIES, part = op % COPIES;
      const uint32_t to = !FP8        ? part * G::KV_BLK + my_box * box * G::SWZ
                          : part == 0 ? my_box * box * D
                                      : KEYS * D + my_box * box * 4;
      uint32_t qe_ph = 0u;   // q_empty
      uint32_t q_par = 1u;   // parity of the last Q load's q_full phase
      bool q_loaded = false;
      constexpr int RING = FP8 ? G::RAW_STAGES : STAGES;
      uint64_t* const full = FP8 ? sh->raw_full : sh->kv_full;
      uint64_t* const empty = FP8 ? sh->raw_empty : sh->kv_empty;
      int slot = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      ProducersMeet<2> meet{sh->issued, 3};
      while (issued < meet.limit && next_part()) {
        // the page of this lane's copies for a tile: its entry is fetched one tile ahead
        const int tile1 = my_box < boxes ? min(w.tile1, (w.s.len - my_box * box + KEYS - 1) / KEYS) : 0;
        auto fetch = [&](int t) -> int {
          return t < tile1 ? page_entry(p.seqs, w.b, t * KEYS + my_box * box) : 0;
        };
        int entry = fetch(w.tile0);
        // The warps load a query tile each.
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          if (!ok || i != pw || (w.steps(p, i) == 0 && !w.paired(p))) continue;
          ok = wait(sh->q_empty[i], qe_ph ^ 1u);
          if (!ok) continue;
          qe_ph ^= 1u;
          q_par ^= 1u;
          q_loaded = true;
          if (lane == 0) {
            const uint32_t bar = smem_u32(&sh->q_full[i]);
            mbar_arrive_expect_tx(bar, p.tile_live * G::ROW_BYTES);
#pragma unroll
            for (int c = 0; c < G::NBLK; ++c)
              tma_load_3d(smem_u32(q_smem + i * G::Q_TILE + c * G::Q_BLK), &tmQ, bar,
                          c * (G::SWZ / 2), w.head * p.group,
                          w.s.first + w.tok0(p, w.paired(p) ? 0 : i));
          }
        }
        bool stop = false;
        for (int t = w.tile0; t < w.tile1 && !stop; ++t) {
          const int key0 = t * KEYS;
          const int page = t < tile1 ? checked_page(p.seqs, entry) : -1;
          entry = fetch(t + 1);
          const int row = (key0 + my_box * box) & (size - 1);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (ok) ok = wait(empty[slot], ph ^ 1u);
            if (!ok) {
              meet(pw, issued);
              stop = issued >= meet.limit;
              if (stop) break;
            }
            const uint32_t bar = smem_u32(&full[slot]);
            if (page >= 0) {
              const CUtensorMap* map = kv ? &tmV : &tmK;
              if constexpr (FP8) {
                const uint32_t dst = smem_u32(raw_smem + slot * G::RAW) + to;
                if (part == 0) {
                  tma_load_4d(dst, map, bar, 0, row, w.head, page);
                } else {
                  const float* src = kv ? p.v_scale + page * p.v_scale_stride[0] + w.head * p.v_scale_stride[1]
                                        : p.k_scale + page * p.k_scale_stride[0] + w.head * p.k_scale_stride[1];
                  bulk_load_tile(dst, src + row, box * 4, bar);
                }
              } else {
                tma_load_4d(smem_u32(kv_smem + slot * G::KV_TILE) + to, map, bar,
                            part * (G::SWZ / 2), row, w.head, page);
              }
            }
            __syncwarp();
            // (as in the row kernel: copies may land before this, and both warps arrive)
            if (lane == 0) {
              const int live = min(boxes, max(0, (w.s.len - key0 + box - 1) / box));  // with a key
              if (pw == 0) mbar_arrive_expect_tx(bar, live * box * (FP8 ? D + 4 : G::ROW_BYTES));
              else mbar_arrive(bar);
            }
            if (!FP8 && kv == 1 && t + 1 == w.tile1 && w.tail() && pw == 0 && lane == 0)
              mbar_arrive(smem_u32(&sh->v_go[slot]));
            ++issued;
            if (++slot == RING) {
              slot = 0;
              ph ^= 1u;
            }
          }
        }
        if (pw == 0 && lane == 0 &&
            (fresh(p.seqs.kv_lens + w.b) != w.s.len ||
             fresh(p.seqs.offsets + w.b + 1) - fresh(p.seqs.offsets + w.b) != w.s.count))
          report(status, kStatusPageTable);
      }
      meet(pw, issued);
      // the copies issued last land before shared memory goes away
      if (q_loaded) drain_bar(smem_u32(&sh->q_full[pw]), q_par);
      for (int u = 0; u < min(issued, RING); ++u) {
        const int x = issued - 1 - u;
        drain_bar(smem_u32(&full[x % RING]), static_cast<uint32_t>((x / RING) & 1));
      }
    } else if (warp == G::MMA_WARP || TILES == 2) {
      // ---------------------------------------------------------------- MMA issuers
      // Tile 0's issuer and tile 1's take turns through two named barriers, per part: S_0, S_1, then
      // per step tile 0's P V and next S, and tile 1's.  Both make every hand-off on every path.
      constexpr uint32_t kTok0 = 1, kTok1 = 2;
      const int ti = warp == G::MMA_WARP ? 0 : 1;
      constexpr uint32_t hi = ((8u * G::SWZ) >> 4) | (1u << 14) | (G::LAYOUT << 29);
      const uint32_t q_lo = (smem_u32(q_smem + ti * G::Q_TILE) >> 4) | (1u << 16);
      const uint32_t k_lo = (smem_u32(kv_smem) >> 4) | (1u << 16);
      const uint32_t v_lo = (smem_u32(kv_smem) >> 4) | (static_cast<uint32_t>(G::KV_BLK >> 4) << 16);
      constexpr uint32_t kSlot = G::KV_TILE >> 4;
      const uint32_t s_bar = smem_u32(&sh->s_full[ti]);
      const uint32_t dS = tmem + ti * KEYS;
      const uint32_t dO = tmem + G::TMEM_O + ti * D;
      const bool lead = lane == 0;
      auto issue_s = [&](int slot) {
        const uint32_t b0 = k_lo + static_cast<uint32_t>(slot) * kSlot;
#pragma unroll
        for (int c = 0; c < G::NBLK; ++c)
#pragma unroll
          for (int k = 0; k < G::SWZ / 32; ++k)
            mma_f16_ss_lo(dS, q_lo + ((c * G::Q_BLK + k * 32) >> 4),
                          b0 + ((c * G::KV_BLK + k * 32) >> 4), hi, IDESC_S, (c | k) ? 1u : 0u);
      };
      auto issue_pv = [&](int slot, uint32_t acc) {
        const uint32_t b0 = v_lo + static_cast<uint32_t>(slot) * kSlot;
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k)
          mma_f16_ts_lo(dO, dS + k * 8, b0 + ((k * 16 * G::SWZ) >> 4), hi, IDESC_O,
                        k > 0 ? 1u : acc);
      };
      auto pass_turn = [&]() {
        __syncwarp();
        if (TILES == 2) named_barrier_arrive(ti == 0 ? kTok0 : kTok1, 64);
      };
      auto take_turn = [&]() {
        __syncwarp();
        if (TILES == 2) named_barrier_sync(ti == 0 ? kTok1 : kTok0, 64);
      };
      uint32_t q_ph = 0, p_ph = 0, oe_ph = 0;
      uint32_t clean_ph = 0;  // bit s: parity of v_clean[s]
      int slot = 0;
      uint32_t ph = 0;
      bool ok = true;
      bool first_turn = true;  // tile 0's very first turn is the only one without a take
      while (next_part()) {
        const int n = w.tile1 - w.tile0;
        const int mine = w.steps(p, ti);
        const bool tail = !FP8 && w.tail();
        if (w.paired(p)) {
          // Both issuers work on the one query tile, on every other key tile each and without
          // turns.  A slot is given back by both: by the one that uses it once its MMAs are done,
          // by the other as soon as the slot is full.
          if (ok) ok = wait(sh->q_full[ti], q_ph);
          q_ph ^= 1u;
          for (int j = 0; j < n; ++j) {
            const bool act = (j & 1) == ti;
            if (ok) ok = wait(sh->kv_full[slot], ph);
            if (ok && lead) {
              if (act) {
                tc_fence_after();
                issue_s(slot);
                mma_commit(s_bar);
                if (j + 2 >= n) mma_commit(smem_u32(&sh->q_empty[ti]));
                mma_commit(smem_u32(&sh->kv_empty[slot]));
              } else {
                mbar_arrive(smem_u32(&sh->kv_empty[slot]));
              }
            }
            if (++slot == STAGES) { slot = 0; ph ^= 1u; }
            if (ok) ok = wait(sh->kv_full[slot], ph);
            if (tail && j + 1 == n) {
              if (ok) ok = wait(sh->v_clean[slot], (clean_ph >> slot) & 1u);
              clean_ph ^= 1u << slot;
            }
            if (act) {
              if (ok) ok = wait(sh->p_ready[ti], p_ph);
              p_ph ^= 1u;
              if (j < 2) {
                if (ok) ok = wait(sh->o_empty[ti], oe_ph ^ 1u);
                oe_ph ^= 1u;
              }
            }
            if (ok && lead) {
              if (act) {
                tc_fence_after();
                issue_pv(slot, j >= 2 ? 1u : 0u);
                if (j + 2 >= n) mma_commit(smem_u32(&sh->o_full[ti]));
                mma_commit(smem_u32(&sh->kv_empty[slot]));
              } else {
                mbar_arrive(smem_u32(&sh->kv_empty[slot]));
              }
            }
            __syncwarp();
            if (++slot == STAGES) { slot = 0; ph ^= 1u; }
          }
          continue;
        }
        const int k0 = slot;
        if (ok) ok = wait(sh->kv_full[slot], ph);
        if (++slot == STAGES) { slot = 0; ph ^= 1u; }
        if (ok && mine > 0) {
          ok = wait(sh->q_full[ti], q_ph);
          q_ph ^= 1u;
        }
        tc_fence_after();
        if (ti == 1 || !first_turn) take_turn();
        first_turn = false;
        if (ok && lead) {
          if (mine > 0) {
            issue_s(k0);
            mma_commit(s_bar);
            if (mine == 1) mma_commit(smem_u32(&sh->q_empty[ti]));
          }
          mma_commit(smem_u32(&sh->kv_empty[k0]));
        }
        pass_turn();
        for (int j = 0; j < n; ++j) {
          const bool act = j < mine;
          const bool s_next = j + 1 < mine;
          const bool k_next = j + 1 < n;
          const int vslot = slot;
          const uint32_t vph = ph;
          if (++slot == STAGES) { slot = 0; ph ^= 1u; }
          const int kslot = slot;
          const uint32_t kph = ph;
          if (k_next && ++slot == STAGES) { slot = 0; ph ^= 1u; }
          if (ok) ok = wait(sh->kv_full[vslot], vph);
          if (tail && !k_next) {
            if (ok) ok = wait(sh->v_clean[vslot], (clean_ph >> vslot) & 1u);
            clean_ph ^= 1u << vslot;
          }
          if (ok && k_next) ok = wait(sh->kv_full[kslot], kph);
          if (ok && act) {
            ok = wait(sh->p_ready[ti], p_ph);
            p_ph ^= 1u;
          }
          if (ok && act && j == 0) {
            ok = wait(sh->o_empty[ti], oe_ph ^ 1u);  // the previous part's output has been read
            oe_ph ^= 1u;
          }
          tc_fence_after();
          take_turn();
          if (ok && lead) {
            if (act) {
              issue_pv(vslot, j > 0 ? 1u : 0u);
              if (s_next) {
                issue_s(kslot);
                mma_commit(s_bar);
                if (j + 2 == mine) mma_commit(smem_u32(&sh->q_empty[ti]));
              } else {
                mma_commit(smem_u32(&sh->o_full[ti]));
              }
            }
            mma_commit(smem_u32(&sh->kv_empty[vslot]));
            if (k_next) mma_commit(smem_u32(&sh->kv_empty[kslot]));
          }
          pass_turn();
        }
      }
      // tile 1's last hand-off (there is none in a CTA without work)
      if (ti == 0 && !first_turn) take_turn();
      if (lead) mma_commit(smem_u32(&sh->mma_done));
      __syncwarp();
      drain_bar(smem_u32(&sh->mma_done), 0);
    }
  } else if (warp >= 8) {
    {
      setmaxnreg_dec<G::REG_AUX>();
      // ------------------------------------------------ the sequence's end, or dequantising
      const int tid = threadIdx.x - 256;
      int slot = 0;
      uint32_t ph = 0;
      bool ok = true;
      if constexpr (!FP8) {
        // These warps take no part in the other tiles, so a slot may go through many fills that
        // they do not see: v_go tells them that the one they clean is under way.  The issuers
        // need v_clean, so neither barrier of a slot can get a second phase ahead.
        uint32_t go_ph = 0;  // bit s: parity of v_go[s]
        while (ok && next_part()) {
          const int n = 2 * (w.tile1 - w.tile0);  // slots of the part; V of the last step is last
          const int last = slot + n - 1;
          const int vslot = last % STAGES;
          const uint32_t vph = ph ^ ((last / STAGES) & 1);
          ph ^= ((slot + n) / STAGES) & 1;
          slot = (slot + n) % STAGES;
          if (!w.tail()) continue;
          ok = wait(sh->v_go[vslot], (go_ph >> vslot) & 1u) && wait(sh->kv_full[vslot], vph);
          go_ph ^= 1u << vslot;
          if (!ok) break;
          const int keep = max(0, w.s.len - (w.tile1 - 1) * KEYS);  // rows of the tile that stay
          constexpr int PIECES = G::SWZ / 16;
          uint8_t* tile = kv_smem + vslot * G::KV_TILE;
          for (int x = tid; x < (KEYS - keep) * PIECES * G::NBLK; x += 128) {
            const int piece = x % PIECES, row = (x / PIECES) % (KEYS - keep) + keep;
            const int c = x / (PIECES * (KEYS - keep));
            *reinterpret_cast<uint4*>(tile + c * G::KV_BLK + row * G::SWZ + piece * 16) =
                make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->v_clean[vslot]));
        }
      } else {
        // A thread takes 16 codes of a row at a time.  The lanes of a warp are LP to a row, and
        // neighbouring rows take different groups of pieces, so that neither the reads of codes
        // nor the writes of operands (two 16-byte chunks, swizzled) meet in a bank.
        int rslot = 0;
        uint32_t rph = 0;
        constexpr int PR = D / 16;                // pieces of a row
        constexpr int LP = PR < 4 ? PR : 4;
        constexpr int RW = 32 / LP;               // rows of a warp at a time
        constexpr int NG = PR / LP;               // groups of pieces
        // rows that the warps take at a time; with short rows not all of them have any
        constexpr int AT_ONCE = G::AUX * RW < KEYS ? G::AUX * RW : KEYS;
        constexpr int STEPS = KEYS / AT_ONCE;
        static_assert(STEPS * AT_ONCE == KEYS, "rows");
        const int row0 = (warp - 8) * RW + lane / LP;
        const int group0 = row0 & (NG - 1);       // groups in an order that differs by row
        static_assert(AT_ONCE % 8 == 0, "the swizzle repeats every 8 rows");
        while (ok && next_part()) {
          for (int t = w.tile0; t < w.tile1 && ok; ++t) {
            const int keep = w.s.len - t * KEYS;
#pragma unroll 1
            for (int kv = 0; kv < 2 && ok; ++kv) {
              ok = wait(sh->raw_full[rslot], rph) && wait(sh->kv_empty[slot], ph ^ 1u);
              if (!ok) break;
              const uint8_t* raw = raw_smem + rslot * G::RAW;
              const float* scale = reinterpret_cast<const float*>(raw + KEYS * D);
              uint8_t* dst = kv_smem + slot * G::KV_TILE;
              // (a branch for each pair of codes took longer than the conversion itself: tail and
              // kind of scale are looked at outside)
              auto piece = [&](int k, int s, auto tail, auto direct, float sc) {
                const int row = row0 + k * AT_ONCE;
                const uint4 code =
                    *reinterpret_cast<const uint4*>(raw + row * D + (group0 ^ s) * LP * 16 + lane % LP * 16);
                const uint32_t cw[4] = {code.x, code.y, code.z, code.w};
                const __half2 hs = __float2half2_rn(sc);
                uint32_t out[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                  const uint32_t h2 = e4m3x2_to_h2(static_cast<uint16_t>(cw[u >> 1] >> (16 * (u & 1))));
                  if constexpr (direct.value) {
                    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h2), hs);
                    out[u] = *reinterpret_cast<const uint32_t*>(&x);
                  } else {
                    const float2 f = fmul2(__half22float2(*reinterpret_cast<const __half2*>(&h2)),
                                           make_float2(sc, sc));
                    out[u] = pack2(f.x, f.y, static_cast<T*>(nullptr));
                  }
                }
                if constexpr (tail.value) {
#pragma unroll
                  for (int u = 0; u < 8; ++u) out[u] = row < keep ? out[u] : 0u;
                }
                const int c = (group0 ^ s) * LP + lane % LP;
                uint8_t* blk = dst + (c * 32 / G::SWZ) * G::KV_BLK;
                const uint32_t at = row0 * G::SWZ + (c * 32) % G::SWZ;  // (AT_ONCE keeps the swizzle)
                uint8_t* to = blk + k * AT_ONCE * G::SWZ;
                *reinterpret_cast<uint4*>(to + swizzle<G::SWZ>(at)) =
                    make_uint4(out[0], out[1], out[2], out[3]);
                *reinterpret_cast<uint4*>(to + swizzle<G::SWZ>(at + 16)) =
                    make_uint4(out[4], out[5], out[6], out[7]);
              };
              auto convert = [&](auto tail) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                  const float sc = scale[row0 + k * AT_ONCE];
                  // a scale that fp16 holds: the product is rounded once either way
                  if (kHalf && __all_sync(0xffffffffu, __half2float(__float2half_rn(sc)) == sc)) {
#pragma unroll
                    for (int s = 0; s < NG; ++s) piece(k, s, tail, std::true_type{}, sc);
                  } else {
#pragma unroll
                    for (int s = 0; s < NG; ++s) piece(k, s, tail, std::false_type{}, sc);
                  }
                }
              };
              if (row0 >= AT_ONCE) {
              } else if (keep >= KEYS) {
                convert(std::false_type{});
              } else {
                convert(std::true_type{});
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(smem_u32(&sh->kv_full[slot]));
                mbar_arrive(smem_u32(&sh->raw_empty[rslot]));
              }
              if (++slot == STAGES) { slot = 0; ph ^= 1u; }
              if (++rslot == G::RAW_STAGES) { rslot = 0; rph ^= 1u; }
            }
          }
        }
      }
    }
  } else {
    setmaxnreg_inc<G::REG_SOFTMAX>();
    const int i = warp >> 2;  // query tile
    if (i < TILES) {
      // ---------------------------------------------------------------- softmax and output
      const int r = threadIdx.x & 127;
      const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t tS = tmem + lane_off + i * KEYS;
      const uint32_t tO = tmem + lane_off + G::TMEM_O + i * D;
      const float sl2 = p.scale_log2;
      const float2 sc = make_float2(sl2, sl2);
      const int r_tok = r / p.group, r_head = r % p.group;  // of the tile
      const bool wide = (reinterpret_cast<uintptr_t>(p.o) | p.o_stride[0] * 2 | p.o_stride[1] * 2) % 32 == 0;
      uint32_t s_ph = 0, of_ph = 0;
      bool ok = true;

      // p = 2^(s * scale + shift), P to TMEM in 32-key chunks; returns the sum of p.  With `upper`
      // the upper half of s is still being loaded, and waited for behind the lower half.
      auto exp_pass = [&](float* s, float m, bool upper) -> float {
        const float shift = (m == -INFINITY ? 0.f : -m) + kPOffset;
        const float2 nm = make_float2(shift, shift);
        float2 acc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < KEYS / 32; ++c) {
          if (c == KEYS / 64 && upper) {
            tmem_wait_ld();
#pragma unroll
            for (int k = KEYS / 2; k < KEYS; ++k) asm volatile("" : "+f"(s[k]));
          }
          uint32_t pk[16];
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const int k = c * 32 + 2 * u;
            const float2 x = ffma2(make_float2(s[k], s[k + 1]), sc, nm);
            const float2 pr = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            acc[u & 3] = fadd2(acc[u & 3], pr);
            pk[u] = pack2(pr.x, pr.y, static_cast<T*>(nullptr));
          }
          tmem_st16(tS + c * 16, pk);
        }
        const float2 a = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
        return a.x + a.y;
      };
      constexpr float kBound = kHalf ? P_SUM_BOUND * 128.f : P_SUM_BOUND;  // 2^P_OFFSET

      // (a wait that gave up does not end the loop: the two sides still meet where they are paired)
      while (next_part()) {
        const bool paired = w.paired(p);
        const int tile = paired ? 0 : i;  // of the block
        // key tiles of this side: first, first + stride, ..
        const int first = paired ? i : 0, stride = paired ? 2 : 1;
        const int n = paired ? (w.tile1 - w.tile0 - i + 1) / 2 : w.steps(p, i);
        const int tok = w.tok0(p, tile) + r_tok;
        const bool live = r < p.tile_live && tok < w.s.count;
        const int64_t row = w.s.first + tok;
        const int head = w.head * p.group + r_head;
        const int64_t part_row = (static_cast<int64_t>(blockIdx.x) * 2 + w.slot()) * (128 * TILES) +
                                 tile * 128 + r;
        const bool whole = w.whole();
        if (threadIdx.x == 0 && !whole && w.slot() == 0) p.parts[blockIdx.x] = w.note(range, p.item_cost);
        if (n == 0) {
          // nothing of this part concerns the tile (no token, or keys behind all of them)
          if (live && !whole) p.part_lse[part_row] = -INFINITY;
          continue;
        }
        const int past = w.s.len - w.s.count;
        const int lim = p.causal ? min(w.s.len, past + tok + 1) : w.s.len;  // keys of this row
        const int lim_all = p.causal ? min(w.s.len, past + w.tok0(p, tile) + 1) : w.s.len;
        const int key_first = (w.tile0 + first) * KEYS;
        float m = -INFINITY;  // the row's base, log2 units
        float l = 0.f;
        float s[KEYS];
        for (int j = 0; j < n && ok; ++j) {
          ok = wait(sh->s_full[i], s_ph);
          if (!ok) break;
          s_ph ^= 1u;
          tc_fence_after();
          const int key0 = key_first + j * stride * KEYS;
          const bool masked = key0 + KEYS > lim_all;
          // the first step and masked ones take the whole row at once
          const bool upper = j > 0 && !masked;
#pragma unroll
          for (int c = 0; c < KEYS / 64; ++c)
            tmem_ld32(tS + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
          if (upper) {
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < KEYS / 2; ++k) asm volatile("" : "+f"(s[k]));
          }
#pragma unroll
          for (int c = KEYS / 64; c < KEYS / 32; ++c)
            tmem_ld32(tS + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
          if (!upper) {
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < KEYS; ++k) asm volatile("" : "+f"(s[k]));
          }
          if (masked) {
            const int keep = lim - key0;
#pragma unroll
            for (int k = 0; k < KEYS; ++k)
              if (k >= keep) s[k] = -INFINITY;
          }
          if (j == 0) {
            m = row_max<KEYS>(s) * sl2;
            l = exp_pass(s, m, false);
          } else {
            float sum = exp_pass(s, m, upper);
            if (__any_sync(0xffffffffu, !(sum <= kBound) || m == -INFINITY)) {
              const float top = row_max<KEYS>(s) * sl2;
              const bool need = top > m + RESCALE_LOG2;
              if (__any_sync(0xffffffffu, need)) {
                float f = 1.f;
                if (need) {
                  f = ex2_approx(m - top);  // m = -inf gives 0
                  m = top;
                }
                l *= f;
                tmem_wait_st();  // the first pass's P lands before it is overwritten
                // O holds the steps before this one: S of this step was issued behind them
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                  uint32_t o[16];
                  tmem_ld16(tO + c * 16, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int u = 0; u < 16; ++u) {
                    asm volatile("" : "+r"(o[u]));
                    o[u] = __float_as_uint(__uint_as_float(o[u]) * f);
                  }
                  tmem_st16(tO + c * 16, o);
                }
                sum = exp_pass(s, m, false);
              }
            }
            l += sum;
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->p_ready[i]));
        }
        if (ok) ok = wait(sh->o_full[i], of_ph);
        of_ph ^= 1u;
        tc_fence_after();
        float w_own = 1.f, w_other = 0.f;  // weights of the two sides' O
        if (paired) {
          sh->pair[i][r] = make_float2(m, l);
          tc_fence_before();
          named_barrier_sync(4, 256);
          tc_fence_after();
          const float2 other = sh->pair[i ^ 1][r];
          const float top = fmaxf(m, other.x);
          w_own = m == top ? 1.f : ex2_approx(m - top);
          w_other = other.x == top ? 1.f : ex2_approx(other.x - top);
          m = top;
          l = l * w_own + other.y * w_other;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        w_own *= inv;
        w_other *= inv;
        __syncwarp();
        if (live && ok && (i == 0 || !paired)) {
          const float lse2 = l == 0.f ? -INFINITY : m + (log2f(l) - kPOffset);
          if (whole) p.lse[row * (p.heads_kv * p.group) + head] = lse2 * kLn2;
          else p.part_lse[part_row] = lse2;
        }
        T* out = static_cast<T*>(p.o) + row * p.o_stride[0] + head * p.o_stride[1];
        float* part = p.part_o + part_row * D;
        const uint32_t tO_other = tmem + lane_off + G::TMEM_O + (i ^ 1) * D;
        // (a pair's sides write every other 16 columns)
#pragma unroll 1
        for (int c = first; c < D / 16 && ok; c += stride) {
          uint32_t o[16];
          float f[16];
          __syncwarp();
          tmem_ld16(tO + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            asm volatile("" : "+r"(o[u]));
            f[u] = __uint_as_float(o[u]) * w_own;
          }
          if (paired) {
            tmem_ld16(tO_other + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              asm volatile("" : "+r"(o[u]));
              f[u] = fmaf(__uint_as_float(o[u]), w_other, f[u]);
            }
          }
          if (live && whole) {
            uint32_t pk[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) pk[u] = pack2(f[2 * u], f[2 * u + 1], static_cast<T*>(nullptr));
            // (lanes are a row apart, so a store takes a cycle a lane: 32 bytes at a time if the
            // layout allows)
            if (wide) {
              st_global_v8(out + c * 16, pk);
            } else {
              *reinterpret_cast<uint4*>(out + c * 16) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
              *reinterpret_cast<uint4*>(out + c * 16 + 8) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
            }
          } else if (live) {
            uint32_t b[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) b[u] = __float_as_uint(f[u]);
            st_global_v8(part + c * 16, b);
            st_global_v8(part + c * 16 + 8, b + 8);
          }
        }
        if (paired) {  // both sides have read both O
          tc_fence_before();
          named_barrier_sync(4, 256);
        }
        __syncwarp();
        tc_fence_before();
        if (lane == 0) mbar_arrive(smem_u32(&sh->o_empty[i]));
      }
    }
  }

  // ---- teardown: every thread arrives here exactly once
  tc_fence_before();
  __syncthreads();
  if (warp == G::MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace fa
