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
// Warps (16-bit 12, float8 20):
//   0-3, 4-7  epilogue of key tile 0, 1
//   8         MMA issuer (owns TMEM)
//   9, 10     TMA producers of K
//   11        TMA producer of Q, and the logsumexps of its rows
//   12-19     float8: convert the key tiles
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

template <int D, bool FP8>
struct WeightsGeo {
  static constexpr int QN = D <= 128 ? 128 : FP8 ? 32 : 64;  // rows of a query tile
  static constexpr int ROW_BYTES = 2 * D;
  static constexpr int SWZ = ROW_BYTES >= 128 ? 128 : ROW_BYTES;
  static constexpr int NBLK = ROW_BYTES / SWZ;
  static constexpr int K_BLK = 128 * SWZ;
  static constexpr int K_TILE = 128 * ROW_BYTES;
  static constexpr int Q_BLK = QN * SWZ;
  static constexpr int Q_TILE = QN * ROW_BYTES;
  static constexpr int RAW = FP8 ? 128 * (D + 4) : 0;  // codes, scales
  static constexpr int K_SLOTS = D == 256 ? 2 : FP8 ? 3 : 4;
  static constexpr int Q_SLOTS = D <= 64 ? 4 : 2;
  static constexpr int L_SLOTS = 4;  // logsumexps of query tiles
  static constexpr int RAW_SLOTS = !FP8 ? 0 : D == 256 ? 1 : 3;
  static constexpr int SHARED = 8192;
  static constexpr int TILES = K_SLOTS * K_TILE + Q_SLOTS * Q_TILE + RAW_SLOTS * RAW;
  // more than half of an SM's shared memory in any case: one CTA per SM, which takes all its TMEM
  static constexpr int SMEM = 1024 + TILES + SHARED > 120 * 1024 ? 1024 + TILES + SHARED : 120 * 1024;
  static constexpr int AUX = FP8 ? 8 : 0;
  static constexpr int THREADS = (12 + AUX) * 32;
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
    seq_rows(p.seqs, b, first, count);
    len = seq_len(p.seqs, b);
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

// (plain data: it lives in shared memory)
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
  __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == n; }
  __device__ __forceinline__ int key0() const { return block * kWeightsBlock; }
  __device__ __forceinline__ int tiles() const { return key0() + 128 < s.len ? 2 : 1; }
  // A step's query tile: its first token, its first head of the group, and its rows.
  __device__ __forceinline__ int tok0(const PagedWeightsParams& p, int t) const {
    return (q0 + t) / p.chunks * p.tile_toks;
  }
  __device__ __forceinline__ int head0(const PagedWeightsParams& p, int t) const {
    return (q0 + t) % p.chunks * p.tile_heads;
  }
  __device__ __forceinline__ int rows(const PagedWeightsParams& p, int t) const {
    return min(s.count - tok0(p, t), p.tile_toks) * min(p.group - head0(p, t), p.tile_heads);
  }
};

template <typename G>
struct WeightsShared {
  uint64_t k_full[G::K_SLOTS], k_empty[G::K_SLOTS];
  uint64_t q_full[G::Q_SLOTS], q_empty[G::Q_SLOTS];
  uint64_t l_full[G::L_SLOTS], l_empty[G::L_SLOTS];
  uint64_t raw_full[4], raw_empty[4];
  uint64_t s_full[2][2], s_empty[2][2];
  uint64_t mma_done;
  int page[4][16];       // of a key tile's boxes, -1: none
  int raw_page[4][16];
  float scale[4][128];   // float8: of a key tile's rows
  alignas(16) float neg_lse[G::L_SLOTS][G::QN];  // -l of a query tile's rows
  int issued[2];
  PagedRange range;
  WeightsWalk first_walk;
  int first_more;
  WeightsWalk walks[20];
  int more[20];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

template <typename T, int D, bool FP8>
__global__ void __launch_bounds__(WeightsGeo<D, FP8>::THREADS, 1)
    paged_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ PagedWeightsParams p) {
  using G = WeightsGeo<D, FP8>;
  using Sh = WeightsShared<G>;
  static_assert(sizeof(Sh) <= G::SHARED, "barrier block");
  constexpr int QN = G::QN, K_SLOTS = G::K_SLOTS, Q_SLOTS = G::Q_SLOTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* k_smem = smem;
  uint8_t* q_smem = k_smem + K_SLOTS * G::K_TILE;
  uint8_t* raw_smem = q_smem + Q_SLOTS * G::Q_TILE;
  Sh* sh = reinterpret_cast<Sh*>(raw_smem + G::RAW_SLOTS * G::RAW);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* const status = p.seqs.status;

  let_next_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < K_SLOTS; ++s) {
      mbar_init(smem_u32(&sh->k_full[s]), FP8 ? G::AUX : 2);
      mbar_init(smem_u32(&sh->k_empty[s]), 1 + 8);  // the MMAs, the epilogue
    }
    for (int s = 0; s < Q_SLOTS; ++s) {
      mbar_init(smem_u32(&sh->q_full[s]), 1);
      mbar_init(smem_u32(&sh->q_empty[s]), 1);
    }
    for (int s = 0; s < G::L_SLOTS; ++s) {
      mbar_init(smem_u32(&sh->l_full[s]), 1);
      mbar_init(smem_u32(&sh->l_empty[s]), 8);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(smem_u32(&sh->raw_full[s]), 2);
      mbar_init(smem_u32(&sh->raw_empty[s]), 8);
      mbar_init(smem_u32(&sh->s_full[s >> 1][s & 1]), 1);
      mbar_init(smem_u32(&sh->s_empty[s >> 1][s & 1]), 4);
    }
    mbar_init(smem_u32(&sh->mma_done), 1);
    sh->abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&sh->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  wait_for_launch_before();
  if (threadIdx.x == 0) p.notes[blockIdx.x].first_cta = -1;
  if (warp == 0) {
    const PagedRange r =
        paged_range(p, [&](int b) { const WeightsSeq s(p, b); return s.per_head * p.heads_kv; });
    if (lane == 0) {
      sh->range = r;
      WeightsWalk x(p, r);
      sh->first_more = x.next(p, r.hi);
      sh->first_walk = x;
    }
  }
  __syncthreads();
  const PagedRange& range = sh->range;

  auto wait = [&](uint64_t& bar, uint32_t parity) {
    const bool ok = wait_bar_flag(&sh->abort_flag, smem_u32(&bar), parity, status);
    return static_cast<bool>(__all_sync(0xffffffffu, ok));
  };
  WeightsWalk& w = sh->walks[warp];
  bool begun = false;
  auto next_part = [&]() -> bool {
    __syncwarp();
    if (lane == 0) {
      WeightsWalk x = begun ? w : sh->first_walk;
      sh->more[warp] = begun ? x.next(p, range.hi) : sh->first_more;
      w = x;
    }
    begun = true;
    __syncwarp();
    return sh->more[warp] != 0;
  };
  // The query tile in use; a lone one stays from item to item of the same sequence and head.
  int q_seq = -1, q_head = -1;
  auto same_q = [&]() { return w.s.qtiles == 1 && q_seq == w.b && q_head == w.head; };
  auto now_q = [&]() {
    q_seq = w.b;
    q_head = w.head;
  };

  if (warp == 9 || warp == 10) {
    // ------------------------------------------------------------------ producers of K
    const int pw = warp - 9;
    const int op = lane * 2 + pw;
    constexpr int COPIES = FP8 ? 2 : G::NBLK;  // of one page
    const int size = 1 << p.seqs.page_log2;
    const int box = min(size, 128);
    const int boxes = 128 / box;
    const int my_box = op / COPIES, part = op % COPIES;
    const uint32_t to = !FP8        ? part * G::K_BLK + my_box * box * G::SWZ
                        : part == 0 ? my_box * box * D
                                    : 128 * D + my_box * box * 4;
    constexpr int RING = FP8 ? G::RAW_SLOTS : K_SLOTS;
    uint64_t* const full = FP8 ? sh->raw_full : sh->k_full;
    uint64_t* const empty = FP8 ? sh->raw_empty : sh->k_empty;
    int(*const pages)[16] = FP8 ? sh->raw_page : sh->page;
    int slot = 0, issued = 0;
    uint32_t ph = 0;
    bool ok = true;
    ProducersMeet<2> meet{sh->issued, 3};
    while (issued < meet.limit && next_part()) {
      const int tiles = w.tiles();
      int entry[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int pos = w.key0() + i * 128 + my_box * box;
        entry[i] = my_box < boxes && pos < w.s.len ? page_entry(p.seqs, w.b, pos) : -1;
      }
      bool stop = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= tiles || stop) continue;
        const int key0 = w.key0() + i * 128;
        const int pos = key0 + my_box * box;
        const bool in = my_box < boxes && pos < w.s.len;
        const int page = in ? checked_page(p.seqs, entry[i]) : -1;
        if (ok) ok = wait(empty[slot], ph ^ 1u);
        if (!ok) {
          meet(pw, issued);
          stop = issued >= meet.limit;
          if (stop) continue;
        }
        const uint32_t bar = smem_u32(&full[slot]);
        // (what is no page is copied from another one, and gets no weight)
        if (my_box < boxes && part == 0) pages[slot][my_box] = in && page == entry[i] ? page : -1;
        if (page >= 0) {
          const int row = pos & (size - 1);
          if constexpr (FP8) {
            const uint32_t dst = smem_u32(raw_smem + slot * G::RAW) + to;
            if (part == 0) tma_load_4d(dst, &tmK, bar, 0, row, w.head, page);
            else
              bulk_load_tile(dst, p.k_scale + page * p.k_scale_stride[0] + w.head * p.k_scale_stride[1] + row,
                             box * 4, bar);
          } else {
            tma_load_4d(smem_u32(k_smem + slot * G::K_TILE) + to, &tmK, bar, part * (G::SWZ / 2), row, w.head,
                        page);
          }
        }
        __syncwarp();
        if (lane == 0) {
          const int live = min(boxes, (w.s.len - key0 + box - 1) / box);  // with a key
          if (pw == 0) mbar_arrive_expect_tx(bar, live * box * (FP8 ? D + 4 : G::ROW_BYTES));
          else mbar_arrive(bar);
        }
        ++issued;
        if (++slot == RING) {
          slot = 0;
          ph ^= 1u;
        }
      }
      if (pw == 0 && lane == 0 &&
          (fresh(p.seqs.kv_lens + w.b) != w.s.len ||
           fresh(p.seqs.offsets + w.b + 1) - fresh(p.seqs.offsets + w.b) != w.s.count))
        report(status, kStatusPageTable);
    }
    meet(pw, issued);
    for (int u = 0; u < min(issued, RING); ++u) {  // the copies issued last land before shared memory goes away
      const int x = issued - 1 - u;
      drain_bar(smem_u32(&full[x % RING]), static_cast<uint32_t>((x / RING) & 1));
    }
  } else if (warp == 11) {
    // ------------------------------------------------------------------ producer of Q
    int slot = 0, lslot = 0, issued = 0;
    uint32_t ph = 0, lph = 0;
    bool ok = true;
    while (ok && next_part()) {
      for (int t = w.t0; t < w.t1 && ok; ++t) {
        if (same_q()) continue;
        now_q();
        const int tok0 = w.tok0(p, t), head0 = w.head0(p, t), rows = w.rows(p, t);
        const int each = min(p.group - head0, p.tile_heads);  // rows of a token
        float neg[QN / 32];
#pragma unroll
        for (int u = 0; u < QN / 32; ++u) {
          const int c = u * 32 + lane;
          neg[u] = -INFINITY;
          if (c < rows) {
            const int tok = c / each;
            const float l = fresh(p.row_lse + static_cast<int64_t>(w.s.first + tok0 + tok) * (p.heads_kv * p.group) +
                                  w.head * p.group + head0 + c - tok * each);
            if (l != -INFINITY) neg[u] = -l * kLog2e;  // (a row without keys gives nothing)
          }
        }
        ok = wait(sh->q_empty[slot], ph ^ 1u) && wait(sh->l_empty[lslot], lph ^ 1u);
        if (!ok) break;
#pragma unroll
        for (int u = 0; u < QN / 32; ++u) sh->neg_lse[lslot][u * 32 + lane] = neg[u];
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&sh->l_full[lslot]));
          const uint32_t bar = smem_u32(&sh->q_full[slot]);
          mbar_arrive_expect_tx(bar, p.tile_toks * p.tile_heads * G::ROW_BYTES);
#pragma unroll
          for (int c = 0; c < G::NBLK; ++c)
            tma_load_3d(smem_u32(q_smem + slot * G::Q_TILE + c * G::Q_BLK), &tmQ, bar, c * (G::SWZ / 2),
                        w.head * p.group + head0, w.s.first + tok0);
        }
        __syncwarp();
        ++issued;
        if (++slot == Q_SLOTS) {
          slot = 0;
          ph ^= 1u;
        }
        if (++lslot == G::L_SLOTS) {
          lslot = 0;
          lph ^= 1u;
        }
      }
    }
    for (int u = 0; u < min(issued, Q_SLOTS); ++u) {
      const int x = issued - 1 - u;
      drain_bar(smem_u32(&sh->q_full[x % Q_SLOTS]), static_cast<uint32_t>((x / Q_SLOTS) & 1));
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr uint32_t hi = ((8u * G::SWZ) >> 4) | (1u << 14) | (G::LAYOUT << 29);
    const uint32_t k_lo = (smem_u32(k_smem) >> 4) | (1u << 16);
    const uint32_t q_lo = (smem_u32(q_smem) >> 4) | (1u << 16);
    int kslot = 0, qslot = -1;
    uint32_t kph = 0, qph = 1;   // (qph: of the slot in use)
    bool held = false;           // a lone query tile's slot is given back when the next one comes
    int buf[2] = {0, 0};
    uint32_t sph[2] = {0, 0};
    bool ok = true;
    while (ok && next_part()) {
      const int tiles = w.tiles();
      int ks[2];
      uint32_t kp[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = kslot;
        kp[i] = kph;
        if (i < tiles && ++kslot == K_SLOTS) {
          kslot = 0;
          kph ^= 1u;
        }
      }
      for (int t = w.t0; t < w.t1 && ok; ++t) {
        if (!same_q()) {
          now_q();
          if (held && lane == 0) mma_commit(smem_u32(&sh->q_empty[qslot]));
          held = w.s.qtiles == 1;
          if (++qslot == Q_SLOTS) qslot = 0;
          if (qslot == 0) qph ^= 1u;
          ok = wait(sh->q_full[qslot], qph);
        }
        const int n = min(QN, (w.rows(p, t) + 15) & ~15);
        const uint32_t idesc = make_idesc(Elt<T>::kFmt, false, 128, 16) - (2u << 17) + (static_cast<uint32_t>(n >> 3) << 17);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i >= tiles || !ok) continue;
          if (t == w.t0) ok = wait(sh->k_full[ks[i]], kp[i]);
          if (ok) ok = wait(sh->s_empty[i][buf[i]], sph[i] ^ 1u);
          if (!ok) continue;
          tc_fence_after();
          if (lane == 0) {
            const uint32_t a0 = k_lo + ((ks[i] * G::K_TILE) >> 4);
            const uint32_t b0 = q_lo + ((qslot * G::Q_TILE) >> 4);
            const uint32_t d = tmem + (i * 2 + buf[i]) * QN;
#pragma unroll
            for (int c = 0; c < G::NBLK; ++c)
#pragma unroll
              for (int k = 0; k < G::SWZ / 32; ++k)
                mma_f16_ss_lo(d, a0 + ((c * G::K_BLK + k * 32) >> 4), b0 + ((c * G::Q_BLK + k * 32) >> 4), hi, idesc,
                              (c | k) ? 1u : 0u);
            mma_commit(smem_u32(&sh->s_full[i][buf[i]]));
            if (t + 1 == w.t1) mma_commit(smem_u32(&sh->k_empty[ks[i]]));
          }
          __syncwarp();
          buf[i] ^= 1;
          if (buf[i] == 0) sph[i] ^= 1u;
        }
        if (ok && !held && lane == 0) mma_commit(smem_u32(&sh->q_empty[qslot]));
        __syncwarp();
      }
    }
    if (lane == 0) mma_commit(smem_u32(&sh->mma_done));
    __syncwarp();
    drain_bar(smem_u32(&sh->mma_done), 0);
  } else if (warp >= 12) {
    if constexpr (FP8) {
      // ---------------------------------------------------------------- convert the key tiles
      // (lanes and pieces as in the tile kernel)
      constexpr int PR = D / 16;
      constexpr int LP = PR < 4 ? PR : 4;
      constexpr int RW = 32 / LP;
      constexpr int NG = PR / LP;
      constexpr int AT_ONCE = G::AUX * RW < 128 ? G::AUX * RW : 128;
      constexpr int STEPS = 128 / AT_ONCE;
      const int row0 = (warp - 12) * RW + lane / LP;
      const int group0 = row0 & (NG - 1);
      const int tid = threadIdx.x - 12 * 32;
      int slot = 0, rslot = 0;
      uint32_t ph = 0, rph = 0;
      bool ok = true;
      while (ok && next_part()) {
        for (int i = 0; i < w.tiles() && ok; ++i) {
          ok = wait(sh->raw_full[rslot], rph) && wait(sh->k_empty[slot], ph ^ 1u);
          if (!ok) break;
          const uint8_t* raw = raw_smem + rslot * G::RAW;
          uint8_t* dst = k_smem + slot * G::K_TILE;
          if (tid < 128) sh->scale[slot][tid] = reinterpret_cast<const float*>(raw + 128 * D)[tid];
          else if (tid < 144) sh->page[slot][tid - 128] = sh->raw_page[rslot][tid - 128];
          if (row0 < AT_ONCE) {
#pragma unroll
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
            mbar_arrive(smem_u32(&sh->k_full[slot]));
            mbar_arrive(smem_u32(&sh->raw_empty[rslot]));
          }
          if (++slot == K_SLOTS) { slot = 0; ph ^= 1u; }
          if (++rslot == G::RAW_SLOTS) { rslot = 0; rph ^= 1u; }
        }
      }
    }
  } else {
    // -------------------------------------------------------------------- epilogue
    const int i = warp >> 2;         // key tile
    const int r = threadIdx.x & 127; // key of the tile
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int size = 1 << p.seqs.page_log2;
    const int box_log2 = min(p.seqs.page_log2, 7);
    int kslot = 0, lslot = -1, buf = 0;
    uint32_t kph = 0, lph = 1, sph = 0;
    bool ok = true;
    while (ok && next_part()) {
      const int tiles = w.tiles();
      const bool mine = i < tiles;
      const int pos = w.key0() + i * 128 + r;
      const int past = w.s.len - w.s.count;
      const bool whole = w.whole();
      float old = 0.f, k2 = p.scale_log2;
      float* place = nullptr;
      // Both tiles' slots are waited for and given back by all warps, though each looks at one: a warp that
      // passed over fills of a slot could take an older fill for its own.
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x >= tiles) continue;
        if (ok) ok = wait(sh->k_full[kslot], kph);
        if (ok) {
          if (x == i) {
            const int page = sh->page[kslot][r >> box_log2];
            if (FP8) k2 *= sh->scale[kslot][r];
            if (whole && pos < w.s.len && page >= 0) {
              place = p.weights + page * p.weights_stride[0] + w.head * p.weights_stride[1] + (pos & (size - 1));
              if (!(p.reset_new && pos >= past)) old = fresh(place);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh->k_empty[kslot]));
        }
        if (++kslot == K_SLOTS) {
          kslot = 0;
          kph ^= 1u;
        }
      }
      const float2 kk = make_float2(k2, k2);
      float2 acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = make_float2(0.f, 0.f);
      for (int t = w.t0; t < w.t1 && ok; ++t) {
        if (!same_q()) {
          now_q();
          if (lslot >= 0 && lane == 0) mbar_arrive(smem_u32(&sh->l_empty[lslot]));
          if (++lslot == G::L_SLOTS) lslot = 0;
          if (lslot == 0) lph ^= 1u;
          ok = wait(sh->l_full[lslot], lph);
        }
        if (!mine || !ok) continue;
        ok = wait(sh->s_full[i][buf], sph);
        if (!ok) break;
        tc_fence_after();
        const int live = w.rows(p, t);
        // columns before `from` are hidden from this key: of tokens that come before it
        const int from = p.causal ? max(0, pos - past - w.tok0(p, t)) * p.group : 0;
        const int from_all = p.causal ? max(0, pos - lane + 31 - past - w.tok0(p, t)) * p.group : 0;
        const int from_any = p.causal ? max(0, pos - lane - past - w.tok0(p, t)) * p.group : 0;
        const uint32_t tS = tmem + lane_off + (i * 2 + buf) * QN;
        const float* neg = sh->neg_lse[lslot];
#pragma unroll 1
        for (int c0 = from_any & ~31; c0 < live; c0 += 32) {
          float s[32];
          tmem_ld32(tS + c0, reinterpret_cast<uint32_t*>(s));
          tmem_wait_ld();
#pragma unroll
          for (int u = 0; u < 32; ++u) asm volatile("" : "+f"(s[u]));
          if (c0 >= from_all && c0 + 32 <= live) {
#pragma unroll
            for (int u = 0; u < 32; u += 4) {
              const float4 l = *reinterpret_cast<const float4*>(neg + c0 + u);
              const float2 x = ffma2(make_float2(s[u], s[u + 1]), kk, make_float2(l.x, l.y));
              const float2 y = ffma2(make_float2(s[u + 2], s[u + 3]), kk, make_float2(l.z, l.w));
              acc[u / 4 & 3] = fadd2(acc[u / 4 & 3], make_float2(ex2_approx(x.x), ex2_approx(x.y)));
              acc[(u / 4 & 3) ^ 1] = fadd2(acc[(u / 4 & 3) ^ 1], make_float2(ex2_approx(y.x), ex2_approx(y.y)));
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
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->s_empty[i][buf]));
        buf ^= 1;
        if (buf == 0) sph ^= 1u;
      }
      if (!mine || !ok) continue;
      const float2 a = fadd2(fadd2(acc[0], acc[1]), fadd2(acc[2], acc[3]));
      const float sum = a.x + a.y;
      if (whole) {
        if (place) *place = old + sum;
      } else {
        const int slot = w.t0 == 0 ? 1 : 0;
        p.parts[(static_cast<int64_t>(blockIdx.x) * 2 + slot) * kWeightsBlock + i * 128 + r] = sum;
        if (threadIdx.x == 0 && slot == 0 && w.t1 == w.n)
          p.notes[blockIdx.x] = PagedWeightsNote{range.cta_of(w.item + p.item_cost), w.b, w.head, w.block};
      }
    }
  }

  // ---- teardown: every thread arrives here exactly once
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
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
