// Paged attention of few query rows per kv head (decode, drafts): bound by reading the cache.
//
// Rows of a block are (token, query head of the group) pairs, 8, 16 or 32 of them, so that every
// key and value is read once for all query heads that share it.  A CTA walks its range of key tiles
// (fa_paged_attn.cuh).  Producer warps look the tile's pages up and bring them with TMA copies (rows
// of at most 128 bytes per copy, swizzled) and, for float8, the rows' scales with bulk copies, into
// a ring of stages that is as deep as shared memory allows: what it has to hide is one memory
// latency at full bandwidth, ~45 KB per SM.  Consumer warps take 16 KN keys of the tile each, with
// an online softmax of their own, and join their (m, l, O) through shared memory at the item's end.
//
// The products are formed transposed, with mma m16n8k16 on register fragments:
//   S^T [16 keys x 8 rows] = K Q^T,   p = 2^(S * scale * log2 e - m),   O^T [16 dims x 8 rows] += V^T P^T
// so that K and V are the 16-row operands and decoding's few query rows fill the 8 columns (keys
// as columns would leave half of a 16-row operand empty).  mma.sync takes ~9 cycles a sub-partition
// here (measured), a warp ~1000 cycles for 16 keys at head_dim 128: 8 warps take in ~65 bytes a
// cycle, and an SM's share of the measured memory bandwidth is 23.
//
// Measured (head_dim 128, 8 kv heads of 4 query heads; the first figure of calls from a graph, the second of
// calls one by one): one new token of 64 sequences, 300,000 in the cache in bf16, pages of 16: 190 to 194 us,
// 6.4 TB/s, what a plain copy reaches; 40 sequences, 410,000 tokens in float8: 140 to 148 us, 5.9 to 6.2 TB/s
// (ncu: DRAM 74 to 80 % of its nominal rate, tensor pipe 17 and 10 %).  One sequence of 131,000 tokens in
// fp16, 4 kv heads of 64: 33 us, 4.1 TB/s, of which start, cut and joining are ~10 us.  Two to eight drafted
// tokens of 16 sequences: 56 us, 4.1 TB/s, bound by the 32-row block's chain of mma.sync and softmax (issue
// slots 30 %, tensor pipe 24 %); in float8 55 us, half the bytes in nearly the same time.  One sequence of 777
// tokens and 16 kv heads: 8.3 us, in which 16 SMs take 7 tiles one after the other.
//
// Float8 caches: codes convert exactly to fp16, so the products run in fp16.  Queries in bf16 are
// scaled per row by a power of two to the top of fp16's range first (exact but for values below 2^-29 of
// the row's largest, which are off by at most 2^-40 of it).  The key scale multiplies S.  The value scale
// multiplies p before it is rounded to fp16, relative to a scale mv that O is kept apart from.  Scales may
// lie far apart (a row of zeros has scale 1), and a ratio of scales must not push p out of fp16's range.  So
// mv follows the tiles, up and down, where a tile's scales are not all within 2^8 below it, and a tile whose
// scales spread over more is taken in turns, each with the keys of one such band (the others' logits are
// -inf in it).  The batch above takes 141 us; where each sequence begins with a row of zeros and the other
// scales are below 2^-8, 145; where every 16th row is one, so that every tile takes two turns, 259.  (A second
// product for the keys left out, instead of a second turn, took the registers of the first: 94 us against 88 for
// groups of 16 heads.)
//
// p in fp16 (fp16 caches, float8 caches) carries the factor 2^kPOffset, which l carries too: fp16
// keeps full precision down to 2^-14, and so p does down to 2^-(14 + kPOffset) of the row's
// largest, over a float8 cache times a ratio of at least 2^-8: down to 2^-16 in any case, and what is below
// that is off by at most 2^-27 of it.  Rounding p to 16 bits costs a relative 2^-8 (bf16) or 2^-11 (fp16)
// per term at most, as much as rounding the output once; l sums the unrounded p.
#pragma once

#include <cfloat>
#include <type_traits>

#include "fa_paged_attn.cuh"

namespace fa {

// ROWS rows of a block: 8 (one column group), 16 (two, in every warp) or 32 (two for each half of the
// warps).
template <int D, bool FP8, int ROWS_>
struct RowsGeo {
  static constexpr int ROWS = ROWS_;
  static constexpr int WN = ROWS >= 16 ? 2 : 1;   // column groups of a warp
  static constexpr int WM = ROWS / (8 * WN);      // row groups
  static constexpr int ROW_BYTES = FP8 ? D : 2 * D;
  static constexpr int SPAN = ROW_BYTES >= 128 ? 128 : ROW_BYTES;  // bytes of a copied row
  static constexpr int NSPAN = ROW_BYTES / SPAN;
  // Consumer warps: 8, or 4 where 256 columns of O and Q take a thread's registers.  WK of them
  // share a row group and split the keys of a tile, 16 KN each.
  static constexpr int NW = D == 256 ? 4 : 8;
  static constexpr int WK = NW / WM;
  static constexpr int KN = WM == 1 && 32 * NW * ROW_BYTES >= 65536 ? 1  // stages of ~64 KB
                            : WM == 2 && FP8 && D <= 32             ? 4  // (see DR)
                                                                    : 2;
  static constexpr int KEYS = 16 * WK * KN;            // of a tile
  static constexpr int TILE = KEYS * ROW_BYTES;        // K or V of a stage
  static constexpr int SCALES = FP8 ? KEYS * 4 : 0;    // K or V scales of a stage
  static constexpr int STAGE = 2 * TILE + 2 * SCALES;  // a multiple of 1024
  // The warps' O are joined in the memory of the item's last stage, DR columns at a time.
  static constexpr int DR = NW * 8 * WN * D * 4 <= STAGE ? D : D / 2;
  static_assert(NW * 8 * WN * DR * 4 <= STAGE && DR >= 16, "joining");
  static constexpr int Q_PITCH = 2 * D + 16;  // bytes; rows of the query block in shared memory
  // With 8 consumer warps of 128 columns the producers give most of their registers away:
  // launched at 168 a thread, 256 * 224 + 128 * 40 <= 384 * 168.
  static constexpr bool SPLIT = NW == 8 && D >= 128;
  static constexpr int REG_LAUNCH = 168, REG_CONSUMER = 224, REG_PRODUCER = 40;
  static_assert(256 * REG_CONSUMER + 128 * REG_PRODUCER <= 384 * REG_LAUNCH, "register split");
  static constexpr int NP = 4;  // producer warps
  static constexpr int THREADS = (NW + NP) * 32;
  static constexpr int COPIES = 2 * NSPAN + (FP8 ? 2 : 0);  // of one page
  static_assert(KEYS / 8 * COPIES <= NP * 32, "a lane for every copy of a tile of smallest pages");
  static constexpr int kMostStages = 8;
  static constexpr int FIXED = 1024 + ROWS * Q_PITCH;
  static constexpr int STAGES = (222 * 1024 - FIXED) / STAGE < kMostStages
                                    ? (222 * 1024 - FIXED) / STAGE
                                    : kMostStages;
  static constexpr int SMEM = FIXED + STAGES * STAGE;
  static_assert(STAGES >= 2, "at least two stages");
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x2(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
               : "=r"(a), "=r"(b)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x2_t(uint32_t addr, uint32_t& a, uint32_t& b) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(a), "=r"(b)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1, __half*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1, __nv_bfloat16*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transposes an 8 x 8 matrix of 16-bit values held as a fragment.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// Untiled bulk copy global -> shared (16-byte addresses and size), counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}

// Byte offset of 16-byte piece `piece` of row `row` in a tile of rows of SPAN bytes, as the TMA
// swizzle of that width lays it out.
template <int SPAN>
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
  const int x = SPAN == 128 ? (row & 7) : SPAN == 64 ? ((row >> 1) & 3) : SPAN == 32 ? ((row >> 2) & 1) : 0;
  return static_cast<uint32_t>(row * SPAN + ((piece ^ x) << 4));
}

constexpr float kRescale = 4.f;  // a row's base moves once its max passes it by 2^4
// Value scales that are taken together, relative to the largest of them, and what is left out of account
// relative to the largest of all (O, kept in units of mv, has to stay within fp32's range).
constexpr uint32_t kBandBits = 8;
constexpr float kBand = 1.f / (1 << kBandBits);
constexpr float kLeastScale = 1.f / (1ull << 40) / (1ull << 40);

// T: type of q and the output (and of a 16-bit cache).  LV: a call behind shared prefixes.
template <typename T, int D, bool FP8, int ROWS, bool LV>
__global__ void __launch_bounds__(RowsGeo<D, FP8, ROWS>::THREADS, 1)
    paged_rows_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedParams<LV> p) {
  using G = RowsGeo<D, FP8, ROWS>;
  using C = std::conditional_t<FP8, __half, T>;  // type of the products
  constexpr bool kHalf = std::is_same_v<C, __half>;
  constexpr float kPOffset = kHalf ? 10.f : 0.f;  // p <= 2^(kPOffset + kRescale) < 65504
  // of a scaled query row (bf16 queries over float8)
  constexpr float kQueryUnit = std::is_same_v<T, __nv_bfloat16> ? 1.f / 32768.f : 1.f;
  constexpr int NW = G::NW, KEYS = G::KEYS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[G::STAGES], s_empty[G::STAGES];
  __shared__ alignas(16) float s_m[ROWS][G::WK], s_l[ROWS][G::WK];
  __shared__ volatile uint32_t s_abort;
  __shared__ int s_issued[G::NP];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem + G::STAGES * G::STAGE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  begin_early(p);
  if (threadIdx.x == 0) {
    for (int s = 0; s < G::STAGES; ++s) {
      mbar_init(smem_u32(&s_full[s]), G::NP);
      mbar_init(smem_u32(&s_empty[s]), NW);
    }
    s_abort = 0u;
    fence_mbar_init();
  }
  __syncthreads();
  begin(p);
  if constexpr (!LV) {  // (behind shared prefixes the join goes by `where` alone)
    if (threadIdx.x == 0) p.parts[blockIdx.x].first_cta = -2;
  }
  const PagedRange range =
      paged_range(p, [&](int b) { return paged_seq<ROWS, KEYS>(p, b).steps; });
  PagedWalk<ROWS, KEYS, PagedParams<LV>> w(p, range);
  int* const status = p.seqs.status;

  if (warp >= NW) {
    if constexpr (G::SPLIT) setmaxnreg_dec<G::REG_PRODUCER>();
    // ------------------------------------------------------------------------ producers
    // Every copy of a tile has a lane of its own, spread over the warps: a warp issues the copies
    // of its lanes one after the other, one in 65 cycles (measured), and pages of 8 or 16 tokens
    // make up to 64 copies a tile.
    const int pw = warp - NW;
    const int op = lane * G::NP + pw;
    const int box = min(1 << p.seqs.page_log2, KEYS);  // rows of one copy
    const int boxes = KEYS / box;
    const int my_box = op / G::COPIES, kind = op % G::COPIES;
    const bool is_scale = kind >= 2 * G::NSPAN;
    const bool is_v = is_scale ? kind == 2 * G::NSPAN + 1 : kind >= G::NSPAN;
    const int span = is_v ? kind - G::NSPAN : kind;
    const CUtensorMap* const map = is_v ? &tmV : &tmK;
    const float* const scales = is_v ? p.v_scale : p.k_scale;
    const int64_t* const scale_stride = is_v ? p.v_scale_stride : p.k_scale_stride;
    const uint32_t to = is_scale ? 2 * G::TILE + (is_v ? G::SCALES : 0) + my_box * box * 4
                                 : (is_v ? G::TILE : 0) + span * KEYS * G::SPAN + my_box * box * G::SPAN;
    int slot = 0, issued = 0;
    uint32_t ph = 0;
    bool ok = true;
    ProducersMeet<G::NP> meet{s_issued, 2};
    while (issued < meet.limit && w.next()) {
      if (pw == 0 && lane == 0) {
        const PagedSeqs& from = seqs_of_line(p, w.b);
        const int b = seq_of_line(p, w.b);
        if (fresh(from.kv_lens + b) != w.s.len || fresh(from.offsets + b + 1) - fresh(from.offsets + b) != w.s.count)
          report(status, kStatusPageTable);
      }
      // the page of this lane's copy for a tile: its entry is fetched one tile ahead
      const int tile1 = my_box < boxes ? min(w.tile1, (w.s.len - my_box * box + KEYS - 1) / KEYS) : 0;
      auto fetch = [&](int t) -> int {
        return t < tile1 ? page_entry(seqs_of_line(p, w.b), seq_of_line(p, w.b), t * KEYS + my_box * box) : 0;
      };
      int entry = fetch(w.tile0);
      for (int t = w.tile0; t < w.tile1; ++t) {
        const int key0 = t * KEYS;
        const int page = t < tile1 ? checked_page(p.seqs, entry) : -1;
        entry = fetch(t + 1);
        if (ok) {
          ok = wait_bar_flag(&s_abort, smem_u32(&s_empty[slot]), ph ^ 1u, status);
          ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok) {
          meet(pw, issued);
          if (issued >= meet.limit) break;
        }
        const uint32_t bar = smem_u32(&s_full[slot]);
        if (page >= 0) {
          const uint32_t dst = smem_u32(smem + slot * G::STAGE) + to;
          const int row = (key0 + my_box * box) & ((1 << p.seqs.page_log2) - 1);
          if (FP8 && is_scale)
            bulk_load(dst, scales + page * scale_stride[0] + w.head * scale_stride[1] + row, box * 4, bar);
          else
            tma_load_4d(dst, map, bar, span * (FP8 ? G::SPAN : G::SPAN / 2), row, w.head, page);
        }
        __syncwarp();
        // (Copies may land before their bytes are announced: the phase waits for all arrivals.  A
        // warp without copies arrives too, so that it cannot fall phases behind.)
        if (lane == 0) {
          const int live = min(boxes, max(0, (w.s.len - key0 + box - 1) / box));  // with a key
          if (pw == 0) mbar_arrive_expect_tx(bar, live * box * (2 * G::ROW_BYTES + (FP8 ? 8 : 0)));
          else mbar_arrive(bar);
        }
        ++issued;
        if (++slot == G::STAGES) {
          slot = 0;
          ph ^= 1u;
        }
      }
    }
    meet(pw, issued);
    // the copies issued last land before shared memory goes away
    for (int u = 0; u < min(issued, G::STAGES); ++u) {
      const int i = issued - 1 - u;
      drain_bar(smem_u32(&s_full[i % G::STAGES]), static_cast<uint32_t>((i / G::STAGES) & 1));
    }
    return;
  }

  // -------------------------------------------------------------------------- consumers
  if constexpr (G::SPLIT) setmaxnreg_inc<G::REG_CONSUMER>();
  constexpr int KN = G::KN, WK = G::WK, WN = G::WN;
  constexpr int KSTEPS = D / 16;
  const int g = lane >> 2, t4 = lane & 3;
  const int wk = warp % WK;
  const int first = warp / WK * 8 * WN;  // the warp's first row of the block
  const int key_w = wk * 16 * KN;        // its first key of a tile
  // fragment addresses: 8 x 8 matrices of 16-byte rows, one row per lane; a: (0, c), (8, c),
  // (0, c+1), (8, c+1) and b: (0, c), (0, c+1), (8, c), (8, c+1)
  const int a_row = key_w + (lane & 15), a_piece = lane >> 4;
  const int b_row = key_w + (lane & 7) + ((lane >> 4) << 3), b_piece = (lane >> 3) & 1;
  auto at = [&](uint32_t tile, int row, int piece) -> uint32_t {
    return tile + (piece * 16 / G::SPAN) * KEYS * G::SPAN +
           swizzled<G::SPAN>(row, piece % (G::SPAN / 16));
  };
  int slot = 0;
  uint32_t ph = 0;
  bool ok = true;
  // The sign of the scale goes to the queries, so that logits grow with S * |scale|; a scale of 0
  // is taken as queries of 0.
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  const uint32_t q_flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;

  while (w.next()) {
    const int rows = w.s.count * p.group;
    const int row0 = w.block * ROWS;
    const int past = w.s.len - w.s.count;  // position of the sequence's first query
    // token and head of a row of the block
    const int tok0 = w.block == 0 ? 0 : row0 / p.group;
    const int head0 = row0 - tok0 * p.group;
    auto tok_of = [&](int r) -> int {  // (exact: the sum is far below 2^16)
      return tok0 + (p.group == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(head0 + r), p.group_inv)));
    };
    // The query block comes through shared memory: as fragments straight from global memory it
    // would cost each warp many scattered requests.
    for (int i = threadIdx.x; i < ROWS * D / 8; i += NW * 32) {
      const int r = i / (D / 8), piece = i % (D / 8);
      const int tok = tok_of(r), h = row0 + r - tok * p.group;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row0 + r < rows && p.scale_log2 != 0.f)
        x = fresh(reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.q) + static_cast<int64_t>(w.s.first + tok) * p.q_stride[0] +
            static_cast<int64_t>(w.head * p.group + h) * p.q_stride[1] + piece * 8));
      *reinterpret_cast<uint4*>(s_q + r * G::Q_PITCH + piece * 16) = x;
    }
    // the row that this thread will write
    constexpr int TPR = NW * 32 / ROWS;  // threads of a row
    const int my_r = threadIdx.x / TPR;
    const bool my_live = row0 + my_r < rows;
    const int my_tok = tok_of(my_r);
    const int64_t my_head = w.head * p.group + row0 + my_r - my_tok * p.group;
    const bool causal = is_causal(p, w.b);
    // this thread's logits belong to rows first + 8 n + 2 t4 + {0, 1}
    int lim[WN][2];       // keys that the row may attend to
    float qs[WN][2];      // factor of the row's logits
#pragma unroll
    for (int n = 0; n < WN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = first + 8 * n + 2 * t4 + e;
        lim[n][e] = causal && row0 + r < rows ? min(w.s.len, past + tok_of(r) + 1) : w.s.len;
        qs[n][e] = scale;
      }
    // keys that every row of the warp may attend to, and that any row may
    const int last = min(rows - row0, first + 8 * WN) - 1;
    const int lim_all = causal ? min(w.s.len, past + tok_of(first) + 1) : w.s.len;
    const int lim_any = last < first ? 0 : causal ? min(w.s.len, past + tok_of(last) + 1) : w.s.len;
    named_barrier_sync(1, NW * 32);
    uint32_t qf[WN][KSTEPS][2];
#pragma unroll
    for (int n = 0; n < WN; ++n) {
      const uint8_t* src = s_q + (first + 8 * n + g) * G::Q_PITCH;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        if constexpr (FP8) {  // columns 16 k + 4 t4 .. + 3: the order in which codes come (below)
          const uint2 x = *reinterpret_cast<const uint2*>(src + (16 * k + 4 * t4) * 2);
          qf[n][k][0] = x.x;
          qf[n][k][1] = x.y;
        } else {
          qf[n][k][0] = *reinterpret_cast<const uint32_t*>(src + (16 * k + 2 * t4) * 2);
          qf[n][k][1] = *reinterpret_cast<const uint32_t*>(src + (16 * k + 8 + 2 * t4) * 2);
        }
      }
      if constexpr (FP8 && std::is_same_v<T, __nv_bfloat16>) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          const float2 a = Cvt16<T>::unpack(qf[n][k][0]), z = Cvt16<T>::unpack(qf[n][k][1]);
          top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(z.x), fabsf(z.y)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(15 - x) brings the row's largest into [2^15, 2^16), the top of fp16's range (the 2^15 go
        // back with the key scales, so that no product leaves fp32's range sooner)
        const int x = min(max(static_cast<int>(__float_as_uint(top) >> 23), 16), 254);
        const float inv = __uint_as_float(static_cast<uint32_t>(254 + 15 - x) << 23);
        const float back = __uint_as_float(static_cast<uint32_t>(x) << 23);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float2 a = Cvt16<T>::unpack(qf[n][k][c]);
            qf[n][k][c] = pack2(a.x * inv, a.y * inv, static_cast<__half*>(nullptr));
          }
        // this lane's fragment is of row g, its logits are of rows 2 t4 and 2 t4 + 1
        // (at least FLT_MIN: a factor of 0 would make NaN of masked logits)
        qs[n][0] = fmaxf(scale * __shfl_sync(0xffffffffu, back, 8 * t4), FLT_MIN);
        qs[n][1] = fmaxf(scale * __shfl_sync(0xffffffffu, back, 8 * t4 + 4), FLT_MIN);
      }
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int c = 0; c < 2; ++c) qf[n][k][c] ^= q_flip;
    }

    float o[KSTEPS][WN][4];
    float m[WN][2], l[WN][2];
    // float8: what O is relative to, its inverse, the largest value scale so far, and the bound below
    // which this tile's are left
    float mv = 0.f, inv_mv = 0.f, top_mv = 0.f, below = INFINITY;
#pragma unroll
    for (int n = 0; n < WN; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < KSTEPS; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[d][n][c] = 0.f;
    }

    for (int t = w.tile0; t < w.tile1; ++t) {
      if (ok) {
        ok = wait_bar_flag(&s_abort, smem_u32(&s_full[slot]), ph, status);
        ok = __all_sync(0xffffffffu, ok);
      }
      const int key0 = t * KEYS + key_w;
      if (ok && key0 < lim_any) {
        const uint32_t kb = smem_u32(smem + slot * G::STAGE);
        const uint32_t vb = kb + G::TILE;
        // ---- S^T = K Q^T, KN tiles of 16 keys: entries (key g, row 2 t4), (g, 2 t4 + 1),
        // (g + 8, ..); two sums each where there is one chain only, as an mma waits ~35 cycles for
        // the last one of its sum
        constexpr int SUMS = KN * WN == 1 && KSTEPS > 1 ? 2 : 1;
        float s[KN][WN][4], s2[4];
#pragma unroll
        for (int kn = 0; kn < KN; ++kn)
#pragma unroll
          for (int n = 0; n < WN; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[kn][n][c] = s2[c] = 0.f;
        if constexpr (FP8) {
          // A lane's 4 codes of a 16-byte piece are columns 4 t4 .. + 3: they serve as the
          // fragment's k = 2 t4, + 1 and 2 t4 + 8, + 9, and the query fragments are laid out alike.
#pragma unroll
          for (int k = 0; k < KSTEPS; k += 2)
#pragma unroll
            for (int kn = 0; kn < KN; ++kn) {
              uint32_t r[4];
              if constexpr (KSTEPS == 1) ldsm_x2(at(kb, a_row + 16 * kn, 0), r[0], r[1]);
              else ldsm_x4(at(kb, a_row + 16 * kn, k + a_piece), r);
#pragma unroll
              for (int u = 0; u < (KSTEPS == 1 ? 1 : 2); ++u) {
                const uint32_t a[4] = {e4m3x2_to_h2(r[2 * u]), e4m3x2_to_h2(r[2 * u + 1]),
                                       e4m3x2_to_h2(r[2 * u] >> 16), e4m3x2_to_h2(r[2 * u + 1] >> 16)};
#pragma unroll
                for (int n = 0; n < WN; ++n)
                  mma16816(SUMS == 2 && u ? s2 : s[kn][n], a, qf[n][k + u][0], qf[n][k + u][1], (C*)nullptr);
              }
            }
        } else {
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
            for (int kn = 0; kn < KN; ++kn) {
              uint32_t r[4];
              ldsm_x4(at(kb, a_row + 16 * kn, 2 * k + a_piece), r);
#pragma unroll
              for (int n = 0; n < WN; ++n)
                mma16816(SUMS == 2 && k % 2 ? s2 : s[kn][n], r, qf[n][k][0], qf[n][k][1], (C*)nullptr);
            }
        }
        // ---- the V fragments are on their way during the softmax.  Float8: after the
        // transposition a register holds keys 2 t4, + 1 at columns 2 g, + 1 of a piece.
        uint32_t vr[KN][KSTEPS][FP8 ? 2 : 4];
#pragma unroll
        for (int kn = 0; kn < KN; ++kn)
#pragma unroll
          for (int d = 0; d < KSTEPS; d += FP8 ? 2 : 1) {
            if constexpr (!FP8) {
              ldsm_x4_t(at(vb, b_row + 16 * kn, 2 * d + b_piece), vr[kn][d]);
            } else if constexpr (KSTEPS == 1) {
              ldsm_x2_t(at(vb, a_row + 16 * kn, 0), vr[kn][0][0], vr[kn][0][1]);
            } else {
              uint32_t r[4];
              ldsm_x4_t(at(vb, a_row + 16 * kn, d + a_piece), r);
              vr[kn][d][0] = r[0];
              vr[kn][d][1] = r[1];
              vr[kn][d + 1][0] = r[2];
              vr[kn][d + 1][1] = r[3];
            }
          }
        if constexpr (SUMS == 2) {
#pragma unroll
          for (int c = 0; c < 4; ++c) s[0][0][c] += s2[c];
        }
        const bool tail = key0 + 16 * KN > w.s.len;
        // ---- scales and mask; this thread's keys are key0 + 16 kn + g + {0, 8}
        float vs[KN][2];
        if constexpr (FP8) {
          const float* sk = reinterpret_cast<const float*>(smem + slot * G::STAGE + 2 * G::TILE) + key_w + g;
          const bool hides = key0 + 16 * KN > lim_any;
          uint32_t far = 0;  // of positive floats the bits are ordered, a step of 1 << 23 a power of two
#pragma unroll
          for (int kn = 0; kn < KN; ++kn)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float ks = sk[16 * kn + 8 * h] * kQueryUnit;
              vs[kn][h] = sk[KEYS + 16 * kn + 8 * h];
              // that of a key which no row attends to does not count (behind the last key it may be
              // any bits)
              if (hides && key0 + 16 * kn + 8 * h + g >= lim_any) vs[kn][h] = 0.f;
              far = max(far, __float_as_uint(mv) - __float_as_uint(vs[kn][h]));  // (above mv: wraps)
#pragma unroll
              for (int n = 0; n < WN; ++n) {
                s[kn][n][2 * h] *= ks;
                s[kn][n][2 * h + 1] *= ks;
              }
            }
          // (A turn that takes up what was left always comes here, whatever the bits of the scales are:
          // it takes the largest below the last turn's bound, so that the bound falls and the turns end.)
          if (__any_sync(0xffffffffu, far > kBandBits << 23 || below != INFINITY)) {
            float top = 0.f;
#pragma unroll
            for (int kn = 0; kn < KN; ++kn)
#pragma unroll
              for (int h = 0; h < 2; ++h) top = vs[kn][h] < below ? fmaxf(top, vs[kn][h]) : top;
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            top_mv = fmaxf(top_mv, top);
            const float to = fmaxf(top, kLeastScale * top_mv);
            if (to > mv || (top > 0.f && to < kBand * mv)) {  // the same in every lane
              const float f = mv / to;
#pragma unroll
              for (int d = 0; d < KSTEPS; ++d)
#pragma unroll
                for (int n = 0; n < WN; ++n)
#pragma unroll
                  for (int c = 0; c < 4; ++c) o[d][n][c] *= f;
              mv = to;
              inv_mv = 1.f / to;
            }
            // the keys of this turn, and whether any are left
            bool more = false;
            const float from = top < kBand * mv ? 0.f : kBand * mv;  // (of the least there is no other turn)
#pragma unroll
            for (int kn = 0; kn < KN; ++kn)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const bool later = vs[kn][h] < from && vs[kn][h] > 0.f;
                more |= later;
                if (later || (below != INFINITY && !(vs[kn][h] > 0.f && vs[kn][h] < below))) {
                  vs[kn][h] = 0.f;
#pragma unroll
                  for (int n = 0; n < WN; ++n) s[kn][n][2 * h] = s[kn][n][2 * h + 1] = -INFINITY;
                }
              }
            below = __any_sync(0xffffffffu, more) ? from : INFINITY;
          }
#pragma unroll
          for (int kn = 0; kn < KN; ++kn)
#pragma unroll
            for (int h = 0; h < 2; ++h) vs[kn][h] *= inv_mv;
        }
        if (key0 + 16 * KN > lim_all) {
#pragma unroll
          for (int kn = 0; kn < KN; ++kn)
#pragma unroll
            for (int n = 0; n < WN; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (key0 + 16 * kn + g + 8 * (c >> 1) >= lim[n][c & 1]) s[kn][n][c] = -INFINITY;
        }
        // ---- online softmax of each row; the base moves by steps
        bool move = false;
        float top[WN][2];
#pragma unroll
        for (int n = 0; n < WN; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(s[0][n][e], s[0][n][2 + e]);
#pragma unroll
            for (int kn = 1; kn < KN; ++kn) x = fmax3(x, s[kn][n][e], s[kn][n][2 + e]);
            top[n][e] = x * qs[n][e];
            move |= top[n][e] > m[n][e] + kRescale;
          }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int n = 0; n < WN; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = top[n][e];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
              const float to = x > m[n][e] + kRescale ? x : m[n][e];
              const float f = m[n][e] == to ? 1.f : ex2_approx(m[n][e] - to);
              m[n][e] = to;
              l[n][e] *= f;
#pragma unroll
              for (int d = 0; d < KSTEPS; ++d) {
                o[d][n][e] *= f;
                o[d][n][2 + e] *= f;
              }
            }
        }
        uint32_t pf[KN][WN][2];  // P^T: keys 2 t4, + 1 (and + 8) of row g
#pragma unroll
        for (int n = 0; n < WN; ++n) {
          const float shift0 = (m[n][0] == -INFINITY ? 0.f : -m[n][0]) + kPOffset;
          const float shift1 = (m[n][1] == -INFINITY ? 0.f : -m[n][1]) + kPOffset;
#pragma unroll
          for (int kn = 0; kn < KN; ++kn)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float a = ex2_approx(fmaf(s[kn][n][2 * h], qs[n][0], shift0));
              float z = ex2_approx(fmaf(s[kn][n][2 * h + 1], qs[n][1], shift1));
              l[n][0] += a;
              l[n][1] += z;
              if constexpr (FP8) {
                a *= vs[kn][h];
                z *= vs[kn][h];
              }
              pf[kn][n][h] = transposed(pack2(a, z, static_cast<C*>(nullptr)));
            }
        }
        // ---- O^T += V^T P^T; what lies behind the sequence's last key may be any bits: it counts
        // as 0
#pragma unroll
        for (int kn = 0; kn < KN; ++kn) {
          uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
          if (tail) {
            const int a = w.s.len - (key0 + 16 * kn + 2 * t4), z = a - 8;
            keep0 = a >= 2 ? 0xffffffffu : a == 1 ? 0xffffu : 0u;
            keep1 = z >= 2 ? 0xffffffffu : z == 1 ? 0xffffu : 0u;
          }
#pragma unroll
          for (int d = 0; d < KSTEPS; ++d) {
            uint32_t a[4];
            if constexpr (FP8) {  // bytes regrouped by column: 2 g in rows g, 2 g + 1 in rows g + 8
              const uint32_t x = __byte_perm(vr[kn][d][0], 0, 0x3120);
              const uint32_t z = __byte_perm(vr[kn][d][1], 0, 0x3120);
              a[0] = e4m3x2_to_h2(x);
              a[1] = e4m3x2_to_h2(x >> 16);
              a[2] = e4m3x2_to_h2(z);
              a[3] = e4m3x2_to_h2(z >> 16);
            } else {
#pragma unroll
              for (int c = 0; c < 4; ++c) a[c] = vr[kn][d][c];
            }
            if (tail) {
              a[0] &= keep0;
              a[1] &= keep0;
              a[2] &= keep1;
              a[3] &= keep1;
            }
#pragma unroll
            for (int n = 0; n < WN; ++n)
              mma16816(o[d][n], a, pf[kn][n][0], pf[kn][n][1], (C*)nullptr);
          }
        }
      }
      if (FP8 && ok && below != INFINITY) {  // once more, with the keys that are left: fewer each time
        --t;
        continue;
      }
      if (t + 1 == w.tile1) break;  // the last stage is kept for joining
      __syncwarp();
      // (a stage is given back only if it was seen full: a second fill on top of one that is still
      // landing would upset the barrier)
      if (ok && lane == 0) mbar_arrive(smem_u32(&s_empty[slot]));
      if (++slot == G::STAGES) {
        slot = 0;
        ph ^= 1u;
      }
    }

    // ---- join the warps' parts and write the rows (the barriers are passed on every path)
#pragma unroll
    for (int n = 0; n < WN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        if (g == 0) {
          s_m[first + 8 * n + 2 * t4 + e][wk] = m[n][e];
          s_l[first + 8 * n + 2 * t4 + e][wk] = l[n][e];
        }
      }
    named_barrier_sync(1, NW * 32);
    const bool whole = w.whole();
    const int64_t part_row = (static_cast<int64_t>(blockIdx.x) * 2 + w.slot()) * ROWS + my_r;
    if constexpr (!LV) {
      if (!whole && w.slot() == 0 && threadIdx.x == 0) p.parts[blockIdx.x] = w.note();
    }
    // the largest base of a row's warps
    auto top_of = [&](int r) -> float {
      float x = -INFINITY;
#pragma unroll
      for (int u = 0; u < WK; u += 4) {
        const float4 v = *reinterpret_cast<const float4*>(&s_m[r][u]);
        x = fmax3(fmax3(x, v.x, v.y), v.z, v.w);
      }
      return x;
    };
    float f[WN][2];  // this warp's weight in its rows
#pragma unroll
    for (int n = 0; n < WN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f[n][e] = m[n][e] == -INFINITY ? 0.f : ex2_approx(m[n][e] - top_of(first + 8 * n + 2 * t4 + e));
        if (FP8) f[n][e] *= mv;
      }
    float* const join = reinterpret_cast<float*>(smem + slot * G::STAGE);
    // column c of row x lies at c ^ turn(x): the rows that are written at once differ in banks
    auto turn = [](int x) { return ((x >> 1) & 3) * 8 & (G::DR - 1); };
    float inv = 0.f;
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += G::DR) {
      if (c0 > 0) named_barrier_sync(1, NW * 32);
#pragma unroll
      for (int n = 0; n < WN; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int x = 8 * n + 2 * t4 + e;
          if (row0 + first + x >= rows) continue;  // decoding uses few of the rows
          float* mine = join + (warp * 8 * WN + x) * G::DR;
#pragma unroll
          for (int d = 0; d < G::DR / 16; ++d) {
            const float(&v)[4] = o[c0 / 16 + d][n];
            if constexpr (FP8) {
              *reinterpret_cast<float2*>(mine + ((16 * d + 2 * g) ^ turn(x))) =
                  make_float2(v[e] * f[n][e], v[2 + e] * f[n][e]);
            } else {
              mine[(16 * d + g) ^ turn(x)] = v[e] * f[n][e];
              mine[(16 * d + 8 + g) ^ turn(x)] = v[2 + e] * f[n][e];
            }
          }
        }
      if (c0 == 0 && my_live) {
        // 1 / l of the thread's row, and its logsumexp
        const float top = top_of(my_r);
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < WK; ++u) {
          const float x = s_m[my_r][u];
          sum += s_l[my_r][u] * (x == -INFINITY ? 1.f : ex2_approx(x - top));  // 1: l is 0, or NaN
        }
        inv = sum == 0.f ? 0.f : 1.f / sum;
        if (threadIdx.x % TPR == 0) {
          const float lse2 = sum == 0.f ? -INFINITY : top + (log2f(sum) - kPOffset);
          const int64_t at = static_cast<int64_t>(w.s.first + my_tok) * p.heads_kv * p.group + my_head;
          if constexpr (LV) {
            if (whole) p.lse[level_row(p, w.b) + at] = lse2;
            if (w.tile0 == 0) p.where[level_row(p, w.b) + at] = w.where(my_r);
          } else if (whole) {
            p.lse[at] = lse2 * kLn2;
          }
          if (!whole) p.part_lse[part_row] = lse2;
        }
      }
      named_barrier_sync(1, NW * 32);
      const int w0 = my_r / (8 * WN) * WK;  // the first warp of the row's group
#pragma unroll
      for (int i = 0; i < (G::DR + TPR * 4 - 1) / (TPR * 4); ++i) {
        const int c = (threadIdx.x % TPR + i * TPR) * 4;
        if (c >= G::DR || !my_live) break;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < WK; ++u) {
          const int x = my_r % (8 * WN);
          const float4 v = *reinterpret_cast<const float4*>(
              join + ((w0 + u) * 8 * WN + x) * G::DR + (c ^ turn(x)));
          a.x += v.x;
          a.y += v.y;
          a.z += v.z;
          a.w += v.w;
        }
        if constexpr (LV) {
          const int64_t at =
              level_row(p, w.b) + static_cast<int64_t>(w.s.first + my_tok) * p.heads_kv * p.group + my_head;
          *reinterpret_cast<float4*>((whole ? p.whole_o + at * D : p.part_o + part_row * D) + c0 + c) =
              make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        } else if (whole)
          *reinterpret_cast<uint2*>(static_cast<T*>(p.o) +
                                    static_cast<int64_t>(w.s.first + my_tok) * p.o_stride[0] +
                                    my_head * p.o_stride[1] + c0 + c) =
              make_uint2(pack2(a.x * inv, a.y * inv, static_cast<T*>(nullptr)),
                         pack2(a.z * inv, a.w * inv, static_cast<T*>(nullptr)));
        else
          *reinterpret_cast<float4*>(p.part_o + part_row * D + c0 + c) =
              make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
      }
    }
    // the stage goes back to the producers, whose copies are ordered behind these accesses
    fence_proxy_async_smem();
    __syncwarp();
    if (ok && lane == 0) mbar_arrive(smem_u32(&s_empty[slot]));
    if (++slot == G::STAGES) {
      slot = 0;
      ph ^= 1u;
    }
  }
  end(p);
}

}  // namespace fa
