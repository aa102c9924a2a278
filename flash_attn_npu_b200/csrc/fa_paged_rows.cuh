// Paged attention of few query rows per kv head (decode, drafts): bound by reading the cache.
//
// Rows of a block are (token, query head of the group) pairs, 16 or 32 of them (WM groups), so
// that every key and value is read once for all query heads that share it.  A CTA walks its range
// of key tiles (fa_paged_attn.cuh).  A producer warp looks the tile's pages up and brings them
// with one TMA copy per page (rows of at most 128 bytes per copy, swizzled) and, for float8, the
// rows' scales with bulk copies, into a ring of stages that is as deep as shared memory allows: what
// it has to hide is one memory latency at full bandwidth, ~45 KB per SM.  NW consumer warps take 16
// keys of the tile each, with an online softmax of their own:
//   S = Q K^T (m16n8k16), p = 2^(S * scale * log2 e - m), O += P V (m16n8k16),
// and join their (m, l, O) through shared memory at the item's end.  The tensor work is far from
// its limit here, so mma.sync on register fragments is enough: at head_dim 128 a warp spends ~500
// cycles on 16 keys (8 KB of 16-bit cache), 8 warps take in ~130 bytes a cycle, and an SM's share
// of the measured memory bandwidth is 23 bytes a cycle.
//
// Float8 caches: codes convert exactly to fp16, so the products run in fp16.  Queries in bf16 are
// scaled per row by a power of two into fp16's range first (exact but for values 2^-24 below the
// row's largest).  The key scale multiplies S.  The value scale multiplies p before it is rounded
// to fp16, relative to the largest scale met so far (mv): O and mv are kept apart.
//
// p in fp16 (fp16 caches, float8 caches) carries the factor 2^kPOffset, which l carries too: fp16
// keeps full precision down to 2^-14, and so p does down to 2^-(14 + kPOffset) of the row's
// largest.  Rounding p to 16 bits costs a relative 2^-9 (bf16) or 2^-12 (fp16) per term, as much
// as rounding the output once; l sums the unrounded p.
#pragma once

#include <type_traits>

#include "fa_paged_attn.cuh"

namespace fa {

// WM: 16-row groups of a block.
template <int D, bool FP8, int WM>
struct RowsGeo {
  static constexpr int ROW_BYTES = FP8 ? D : 2 * D;
  static constexpr int SPAN = ROW_BYTES >= 128 ? 128 : ROW_BYTES;  // bytes of a copied row
  static constexpr int NSPAN = ROW_BYTES / SPAN;
  // Consumer warps: 8, or 4 where 256 columns of O and Q take a thread's 255 registers.  WK of
  // them share a row group and split the keys of a tile, 16 KN each.
  static constexpr int NW = D == 256 ? 4 : 8;
  static constexpr int WK = NW / WM;
  static constexpr int KN = WM == 1 && 32 * NW * ROW_BYTES >= 65536 ? 1 : 2;  // stages of ~64 KB
  static constexpr int KEYS = 16 * WK * KN;            // of a tile
  static constexpr int ROWS = 16 * WM;
  static constexpr int TILE = KEYS * ROW_BYTES;        // K or V of a stage
  static constexpr int SCALES = FP8 ? KEYS * 4 : 0;    // K or V scales of a stage
  static constexpr int STAGE = 2 * TILE + 2 * SCALES;  // a multiple of 1024
  static constexpr int GROUP_COLS = D < 32 ? D : 32;   // columns joined at a time
  static constexpr int JOIN_PITCH = GROUP_COLS + 4;
  static constexpr int JOIN = NW * 16 * JOIN_PITCH * 4;
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
  static constexpr int FIXED = 1024 + JOIN;
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

// T: type of q and the output (and of a 16-bit cache).
template <typename T, int D, bool FP8, int WM>
__global__ void __launch_bounds__(RowsGeo<D, FP8, WM>::THREADS, 1)
    paged_rows_kernel(const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const PagedAttnParams p) {
  using G = RowsGeo<D, FP8, WM>;
  using C = std::conditional_t<FP8, __half, T>;  // type of the products
  constexpr bool kHalf = std::is_same_v<C, __half>;
  constexpr float kPOffset = kHalf ? 10.f : 0.f;  // p <= 2^(kPOffset + kRescale) < 65504
  constexpr int NW = G::NW, KEYS = G::KEYS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[G::STAGES], s_empty[G::STAGES];
  __shared__ int64_t s_scratch[40];
  __shared__ float s_m[NW][16], s_l[NW][16];
  __shared__ volatile uint32_t s_abort;
  __shared__ int s_issued[G::NP];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* s_join = reinterpret_cast<float*>(smem + G::STAGES * G::STAGE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The combine kernel may be brought up while this one runs; it waits for its end.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < G::STAGES; ++s) {
      mbar_init(smem_u32(&s_full[s]), 1);
      mbar_init(smem_u32(&s_empty[s]), NW);
    }
    s_abort = 0u;
    fence_mbar_init();
    p.parts[blockIdx.x].first_cta = -2;
  }
  const PagedRange range = paged_range(
      p, s_scratch, [&](int b) { return paged_seq<G::ROWS, KEYS>(p, b).steps; });
  __syncthreads();
  PagedWalk<G::ROWS, KEYS> w(p, range);
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
        if (__ldg(p.seqs.kv_lens + w.b) != w.s.len ||
            __ldg(p.seqs.offsets + w.b + 1) - __ldg(p.seqs.offsets + w.b) != w.s.count)
          report(status, kStatusPageTable);
      }
      // the page of this lane's copy for a tile; looked up one tile ahead
      auto look_up = [&](int t) -> int {
        const int key = t * KEYS + my_box * box;
        if (my_box >= boxes || t >= w.tile1 || key >= w.s.len) return -1;
        const int page = page_of(p.seqs, w.b, key);
        if (page < 0) report(status, kStatusPageTable);
        return max(page, 0);
      };
      int next_page = look_up(w.tile0);
      for (int t = w.tile0; t < w.tile1; ++t) {
        const int key0 = t * KEYS;
        const int page = next_page;
        next_page = look_up(t + 1);
        if (ok) {
          ok = wait_bar_flag(&s_abort, smem_u32(&s_empty[slot]), ph ^ 1u, status);
          ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok) {
          meet(pw, issued);
          if (issued >= meet.limit) break;
        }
        const uint32_t bar = smem_u32(&s_full[slot]);
        // (the other warps' copies may land before this arrival: the phase waits for it)
        if (pw == 0 && lane == 0) {
          const int live = min(boxes, max(0, (w.s.len - key0 + box - 1) / box));  // with a key
          mbar_arrive_expect_tx(bar, live * box * (2 * G::ROW_BYTES + (FP8 ? 8 : 0)));
        }
        __syncwarp();
        if (page >= 0) {
          const uint32_t dst = smem_u32(smem + slot * G::STAGE) + to;
          const int row = (key0 + my_box * box) & ((1 << p.seqs.page_log2) - 1);
          if (FP8 && is_scale)
            bulk_load(dst, scales + page * scale_stride[0] + w.head * scale_stride[1] + row, box * 4, bar);
          else
            tma_load_4d(dst, map, bar, span * (FP8 ? G::SPAN : G::SPAN / 2), row, w.head, page);
        }
        __syncwarp();
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
  constexpr int KN = G::KN, WK = G::WK;
  const int g = lane >> 2, t4 = lane & 3;
  const int wm = warp / WK;                 // row group
  const int key_w = (warp % WK) * 16 * KN;  // this warp's keys of a tile
  constexpr int KSTEPS = D / 16;
  constexpr int NT = D / 8;
  // fragment addresses: matrices of 8 rows x 16 bytes, one row per lane
  const int k_row = key_w + (lane & 7) + ((lane >> 4) << 3);  // K: matrices (n, c), (n, c+1), (n+8, c), ..
  const int k_piece = (lane >> 3) & 1;
  const int v_row = key_w + (lane & 15);                      // V: matrices (k, c), (k+8, c), (k, c+1), ..
  const int v_piece = lane >> 4;
  int slot = 0;
  uint32_t ph = 0;
  bool ok = true;
  // The sign of the scale goes to the queries, so that logits grow with S * |scale|; a scale of 0
  // is taken as queries of 0.
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  const uint32_t q_flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;

  while (w.next()) {
    const int rows = w.s.count * p.group;
    const int row0 = w.block * G::ROWS;
    const int past = w.s.len - w.s.count;  // position of the sequence's first query
    // this thread's rows: g and g + 8 of its group
    int lim[2];       // keys that the row may attend to
    float qs[2];      // factor of the row's logits
    uint32_t qf[KSTEPS][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = row0 + wm * 16 + e * 8 + g;
      const int tok = r / p.group;
      const int h = r - tok * p.group;
      const bool live = r < rows;
      lim[e] = p.causal && live ? min(w.s.len, past + tok + 1) : w.s.len;
      qs[e] = scale;
      const T* src = static_cast<const T*>(p.q) + static_cast<int64_t>(w.s.first + tok) * p.q_stride[0] +
                     static_cast<int64_t>(w.head * p.group + h) * p.q_stride[1];
      const bool load = live && p.scale_log2 != 0.f;
      uint32_t lo[KSTEPS], hi[KSTEPS];
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        if (FP8) {  // columns 16 k + 4 t4 .. + 3: the order in which codes come (below)
          const uint2 x = load ? __ldg(reinterpret_cast<const uint2*>(src + 16 * k + 4 * t4))
                               : make_uint2(0, 0);
          lo[k] = x.x;
          hi[k] = x.y;
        } else {
          lo[k] = load ? __ldg(reinterpret_cast<const unsigned*>(src + 16 * k + 2 * t4)) : 0u;
          hi[k] = load ? __ldg(reinterpret_cast<const unsigned*>(src + 16 * k + 8 + 2 * t4)) : 0u;
        }
      }
      if constexpr (FP8 && std::is_same_v<T, __nv_bfloat16>) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          const float2 a = Cvt16<T>::unpack(lo[k]), z = Cvt16<T>::unpack(hi[k]);
          top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(z.x), fabsf(z.y)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-x brings the row's largest into [1, 2)
        const int x = min(max(static_cast<int>(__float_as_uint(top) >> 23), 2), 252);
        const float inv = __uint_as_float(static_cast<uint32_t>(254 - x) << 23);
        qs[e] = scale * __uint_as_float(static_cast<uint32_t>(x) << 23);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          const float2 a = Cvt16<T>::unpack(lo[k]), z = Cvt16<T>::unpack(hi[k]);
          lo[k] = pack2(a.x * inv, a.y * inv, static_cast<__half*>(nullptr));
          hi[k] = pack2(z.x * inv, z.y * inv, static_cast<__half*>(nullptr));
        }
      }
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        qf[k][e] = lo[k] ^ q_flip;
        qf[k][2 + e] = hi[k] ^ q_flip;
      }
    }
    // keys that every row of the group may attend to, and that any row may
    const int first_row = row0 + wm * 16, last_row = min(rows, first_row + 16) - 1;
    const int lim_all = p.causal ? min(w.s.len, past + first_row / p.group + 1) : w.s.len;
    const int lim_any = first_row >= rows ? 0
                        : p.causal        ? min(w.s.len, past + last_row / p.group + 1)
                                          : w.s.len;

    float o[NT][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float mv = 0.f, inv_mv = 0.f;  // float8: largest value scale so far, and its inverse
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[n][c] = 0.f;

    for (int t = w.tile0; t < w.tile1; ++t) {
      if (ok) {
        ok = wait_bar_flag(&s_abort, smem_u32(&s_full[slot]), ph, status);
        ok = __all_sync(0xffffffffu, ok);
      }
      const int key0 = t * KEYS + key_w;
      if (ok && key0 < lim_any) {
        const uint32_t kb = smem_u32(smem + slot * G::STAGE);
        const uint32_t vb = kb + G::TILE;
        // ---- S = Q K^T: 2 KN tiles of 8 keys
        float s[2 * KN][4];
#pragma unroll
        for (int n = 0; n < 2 * KN; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[n][c] = 0.f;
        if constexpr (FP8) {
          // a lane's 4 codes of a 16-byte piece are columns 4 t4 .. + 3: they serve as the
          // fragment's k = 2 t4, + 1 and 2 t4 + 8, + 9, and the query fragments are laid out alike
          if constexpr (KSTEPS == 1) {
#pragma unroll
            for (int kn = 0; kn < KN; ++kn) {
              uint32_t a, z;
              ldsm_x2(kb + swizzled<G::SPAN>(key_w + 16 * kn + (lane & 15), 0), a, z);
              mma16816(s[2 * kn], qf[0], e4m3x2_to_h2(a), e4m3x2_to_h2(a >> 16), (C*)nullptr);
              mma16816(s[2 * kn + 1], qf[0], e4m3x2_to_h2(z), e4m3x2_to_h2(z >> 16), (C*)nullptr);
            }
          } else {
#pragma unroll
            for (int k = 0; k < KSTEPS; k += 2) {
              const int piece = k + k_piece;
#pragma unroll
              for (int kn = 0; kn < KN; ++kn) {
                uint32_t r[4];
                ldsm_x4(kb + (piece * 16 / G::SPAN) * KEYS * G::SPAN +
                            swizzled<G::SPAN>(k_row + 16 * kn, piece % (G::SPAN / 16)),
                        r);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                  mma16816(s[2 * kn + (u >> 1)], qf[k + (u & 1)], e4m3x2_to_h2(r[u]),
                           e4m3x2_to_h2(r[u] >> 16), (C*)nullptr);
              }
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            const int piece = 2 * k + k_piece;
#pragma unroll
            for (int kn = 0; kn < KN; ++kn) {
              uint32_t r[4];
              ldsm_x4(kb + (piece * 16 / G::SPAN) * KEYS * G::SPAN +
                          swizzled<G::SPAN>(k_row + 16 * kn, piece % (G::SPAN / 16)),
                      r);
              mma16816(s[2 * kn], qf[k], r[0], r[1], (C*)nullptr);
              mma16816(s[2 * kn + 1], qf[k], r[2], r[3], (C*)nullptr);
            }
          }
        }
        // ---- scales and mask; this thread's keys are key0 + 8 n + 2 t4 + {0, 1}
        float2 vs[2 * KN];
        if constexpr (FP8) {
          const float* sk = reinterpret_cast<const float*>(smem + slot * G::STAGE + 2 * G::TILE) +
                            key_w + 2 * t4;
          float top = 0.f;
#pragma unroll
          for (int n = 0; n < 2 * KN; ++n) {
            const float2 ks = *reinterpret_cast<const float2*>(sk + 8 * n);
            vs[n] = *reinterpret_cast<const float2*>(sk + KEYS + 8 * n);
            s[n][0] *= ks.x;
            s[n][1] *= ks.y;
            s[n][2] *= ks.x;
            s[n][3] *= ks.y;
          }
          if (key0 + 16 * KN > w.s.len) {  // a scale behind the last key may be any bits
#pragma unroll
            for (int n = 0; n < 2 * KN; ++n) {
              const int k = key0 + 8 * n + 2 * t4;
              vs[n].x = k < w.s.len ? vs[n].x : 0.f;
              vs[n].y = k + 1 < w.s.len ? vs[n].y : 0.f;
            }
          }
#pragma unroll
          for (int n = 0; n < 2 * KN; ++n) top = fmax3(top, vs[n].x, vs[n].y);
          if (__any_sync(0xffffffffu, top > mv)) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float f = mv / top;  // the same in every lane
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[n][c] *= f;
            mv = top;
            inv_mv = 1.f / top;
          }
#pragma unroll
          for (int n = 0; n < 2 * KN; ++n) {
            vs[n].x *= inv_mv;
            vs[n].y *= inv_mv;
          }
        }
        if (key0 + 16 * KN > lim_all) {
#pragma unroll
          for (int n = 0; n < 2 * KN; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (key0 + 8 * n + 2 * t4 + (c & 1) >= lim[c >> 1]) s[n][c] = -INFINITY;
        }
        // ---- online softmax of each row; the base moves by steps
        float top[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[0][2 * e], s[0][2 * e + 1]);
#pragma unroll
          for (int n = 1; n < 2 * KN; ++n) x = fmax3(x, s[n][2 * e], s[n][2 * e + 1]);
          top[e] = x * qs[e];
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + kRescale || top[1] > m[1] + kRescale)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            const float to = x > m[e] + kRescale ? x : m[e];
            const float f = m[e] == to ? 1.f : ex2_approx(m[e] - to);
            m[e] = to;
            l[e] *= f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              o[n][2 * e] *= f;
              o[n][2 * e + 1] *= f;
            }
          }
        }
        uint32_t pf[KN][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float shift = (m[e] == -INFINITY ? 0.f : -m[e]) + kPOffset;
#pragma unroll
          for (int n = 0; n < 2 * KN; ++n) {
            float a = ex2_approx(fmaf(s[n][2 * e], qs[e], shift));
            float z = ex2_approx(fmaf(s[n][2 * e + 1], qs[e], shift));
            l[e] += a + z;
            if constexpr (FP8) {
              a *= vs[n].x;
              z *= vs[n].y;
            }
            pf[n >> 1][2 * (n & 1) + e] = pack2(a, z, static_cast<C*>(nullptr));
          }
        }
        // ---- O += P V; what lies behind the sequence's last key may be any bits: it counts as 0
        const bool tail = key0 + 16 * KN > w.s.len;
#pragma unroll
        for (int kn = 0; kn < KN; ++kn) {
          uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
          if (tail) {
            const int a = w.s.len - (key0 + 16 * kn + 2 * t4), z = a - 8;
            keep0 = a >= 2 ? 0xffffffffu : a == 1 ? 0xffffu : 0u;
            keep1 = z >= 2 ? 0xffffffffu : z == 1 ? 0xffffu : 0u;
          }
          if constexpr (FP8) {
            // after the transposition a register holds keys 2 t4, + 1 at columns 2 g, + 1 of the
            // piece; its bytes regrouped give the fragments of the even and the odd columns
#pragma unroll
            for (int c = 0; c < KSTEPS; c += 2) {
              uint32_t r[4];
              if constexpr (KSTEPS == 1) {
                ldsm_x2_t(vb + swizzled<G::SPAN>(v_row + 16 * kn, 0), r[0], r[1]);
                r[2] = r[3] = 0;
              } else {
                const int piece = c + v_piece;
                ldsm_x4_t(vb + (piece * 16 / G::SPAN) * KEYS * G::SPAN +
                              swizzled<G::SPAN>(v_row + 16 * kn, piece % (G::SPAN / 16)),
                          r);
              }
#pragma unroll
              for (int u = 0; u < (KSTEPS == 1 ? 1 : 2); ++u) {
                const uint32_t a = __byte_perm(r[2 * u], 0, 0x3120);
                const uint32_t z = __byte_perm(r[2 * u + 1], 0, 0x3120);
                uint32_t e0 = e4m3x2_to_h2(a), e1 = e4m3x2_to_h2(z);
                uint32_t d0 = e4m3x2_to_h2(a >> 16), d1 = e4m3x2_to_h2(z >> 16);
                if (tail) {
                  e0 &= keep0;
                  d0 &= keep0;
                  e1 &= keep1;
                  d1 &= keep1;
                }
                mma16816(o[2 * (c + u)], pf[kn], e0, e1, (C*)nullptr);
                mma16816(o[2 * (c + u) + 1], pf[kn], d0, d1, (C*)nullptr);
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < KSTEPS; ++c) {
              uint32_t r[4];
              const int piece = 2 * c + v_piece;
              ldsm_x4_t(vb + (piece * 16 / G::SPAN) * KEYS * G::SPAN +
                            swizzled<G::SPAN>(v_row + 16 * kn, piece % (G::SPAN / 16)),
                        r);
              if (tail) {
                r[0] &= keep0;
                r[1] &= keep1;
                r[2] &= keep0;
                r[3] &= keep1;
              }
              mma16816(o[2 * c], pf[kn], r[0], r[1], (C*)nullptr);
              mma16816(o[2 * c + 1], pf[kn], r[2], r[3], (C*)nullptr);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s_empty[slot]));
      if (++slot == G::STAGES) {
        slot = 0;
        ph ^= 1u;
      }
    }

    // ---- join the warps' parts and write the rows (the barriers are passed on every path)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (t4 == 0) {
        s_m[warp][e * 8 + g] = m[e];
        s_l[warp][e * 8 + g] = l[e];
      }
    }
    named_barrier_sync(1, NW * 32);
    const bool whole = w.whole();
    const int64_t part_row = (static_cast<int64_t>(blockIdx.x) * 2 + w.slot()) * G::ROWS;
    if (!whole && w.slot() == 0 && threadIdx.x == 0) p.parts[blockIdx.x] = w.note();
    float f[2];  // this warp's weight in its rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < WK; ++u) top = fmaxf(top, s_m[wm * WK + u][e * 8 + g]);
      f[e] = m[e] == -INFINITY ? 0.f : ex2_approx(m[e] - top);
      if (FP8) f[e] *= mv;
    }
    // the row that this thread writes, and 1 / l of it
    constexpr int TPR = NW * 32 / G::ROWS;  // threads of a row
    const int r = threadIdx.x / TPR;
    const int w0 = r / 16 * WK;             // the first warp of its group
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int u = 0; u < WK; ++u) top = fmaxf(top, s_m[w0 + u][r % 16]);
#pragma unroll
    for (int u = 0; u < WK; ++u) {
      const float x = s_m[w0 + u][r % 16];
      sum += s_l[w0 + u][r % 16] * (x == -INFINITY ? 1.f : ex2_approx(x - top));  // 1: l is 0, or NaN
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int row = row0 + r;
    const bool live = row < rows;
    const int64_t tok = w.s.first + row / p.group;
    const int64_t h = w.head * p.group + row % p.group;
    if (live && threadIdx.x % TPR == 0) {
      const float lse2 = sum == 0.f ? -INFINITY : top + (log2f(sum) - kPOffset);
      if (whole) p.lse[tok * p.heads_kv * p.group + h] = lse2 * kLn2;
      else p.part_lse[part_row + r] = lse2;
    }
    T* out = static_cast<T*>(p.o) + tok * p.o_stride[0] + h * p.o_stride[1];
    float* part = p.part_o + (part_row + r) * D;
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += G::GROUP_COLS) {
      float* mine = s_join + warp * 16 * G::JOIN_PITCH;
      if constexpr (FP8) {
#pragma unroll
        for (int c = 0; c < G::GROUP_COLS / 16; ++c) {
          const int n = 2 * (c0 / 16 + c);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float4*>(mine + (e * 8 + g) * G::JOIN_PITCH + 16 * c + 4 * t4) =
                make_float4(o[n][2 * e] * f[e], o[n + 1][2 * e] * f[e],
                            o[n][2 * e + 1] * f[e], o[n + 1][2 * e + 1] * f[e]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < G::GROUP_COLS / 8; ++c) {
          const int n = c0 / 8 + c;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float2*>(mine + (e * 8 + g) * G::JOIN_PITCH + 8 * c + 2 * t4) =
                make_float2(o[n][2 * e] * f[e], o[n][2 * e + 1] * f[e]);
        }
      }
      named_barrier_sync(1, NW * 32);
      for (int c = (threadIdx.x % TPR) * 2; c < G::GROUP_COLS; c += TPR * 2) {
        float a = 0.f, z = 0.f;
#pragma unroll
        for (int u = 0; u < WK; ++u) {
          const float2 x = *reinterpret_cast<const float2*>(s_join + ((w0 + u) * 16 + r % 16) * G::JOIN_PITCH + c);
          a += x.x;
          z += x.y;
        }
        if (live) {
          if (whole)
            *reinterpret_cast<uint32_t*>(out + c0 + c) = pack2(a * inv, z * inv, static_cast<T*>(nullptr));
          else
            *reinterpret_cast<float2*>(part + c0 + c) = make_float2(a * inv, z * inv);
        }
      }
      named_barrier_sync(1, NW * 32);
    }
  }
}

}  // namespace fa
