// Writing packed rows of new tokens into the paged key/value cache, and reading rows back
// (declared in include/fa_paged_sm100.h).
//
// A row is one (token, kv head) of K or V: head_dim values.  Float8 rows are quantised by
//   s = 2^e, e = min{ e >= -126 : max |x| <= 448 * 2^e },   c = round_e4m3(x / s).
// A power of two costs e4m3 nothing (a floating-point format keeps its relative step at any
// magnitude; only rows that spread over more than 2^14 reach its subnormals), makes x / s, c * s
// and the scale itself exact, and leaves the one rounding to 4 bits.
//
// Both directions are bound by memory: each value is read and written once, a thread's piece being 16
// bytes of a 16-bit row or 16 codes of a float8 row (32 bytes of the packed one), head_dim / PIECE
// threads to a row, so that a row's largest magnitude is a few shuffles.  Each CTA takes a run of
// tokens, whose sequences and pages its warps look up (a 32-way search of the offsets).  A write has
// its packed rows on their way before that; a read cannot.  What hides the lookups, and the loads
// where a CTA starts, are other CTAs: two pieces a thread and six (write) or eight (read) CTAs to an
// SM took 24.4 and 61 us where four pieces and four CTAs took 25.3 and 65 (9 prompts of 16700 tokens
// in all, 8 heads of 128, to float8; 56700 tokens back to bf16); one piece and eight: 25.1 and 72.
// (From a graph; 24.7 and 66 called one by one.)  These are 4.2 and 5.5 TB/s, where a plain copy reaches 6.5.  3 us
// of the shorter one is what a call of 16 tokens takes; the rest is that no CTA has its next run's rows on
// their way (issue slots 65 %).
#include <cmath>

#include "../../include/fa_paged_sm100.h"
#include "fa_paged_host.h"
#include "fa_paged_launch.h"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 64;  // tokens of one CTA's run
constexpr int kUnroll = 2;      // pieces of a thread in flight

struct CopyParams {
  PagedSeqs seqs;
  void* cache[2];    // K, V
  float* scale[2];
  void* rows[2];
  int64_t cache_stride[2][3];
  int64_t scale_stride[2][2];
  int64_t row_stride[2][2];
  int heads;
  int head_dim;
  int tokens;           // per CTA
  int lanes_log2;       // pieces of a row
  uint32_t pieces_inv;  // floor(2^32 / pieces of a token) + 1; 0 for a run of one token
};

// Smallest b with offsets[b + 1] > t, by the whole warp (seqs - 1 if there is none).
__device__ __forceinline__ int find_seq(const PagedSeqs& s, int t, int lane) {
  int lo = 0, hi = s.seqs - 1;  // the answer lies in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int probe = min(lo + (lane + 1) * step, hi);  // is the answer >= probe?
    const bool past = fresh(s.offsets + probe) <= t;
    const int n = __popc(__ballot_sync(0xffffffffu, past));
    const int next = min(lo + n * step, hi);
    hi = n == 32 ? hi : min(lo + (n + 1) * step, hi) - 1;
    lo = next;
    hi = max(hi, lo);
  }
  return lo;
}

// Elements of a piece.
template <bool FP8>
constexpr int kPiece = FP8 ? 16 : 8;

// T: type of the packed rows.  FP8: the cache holds e4m3 codes and scales, else T.  WRITE: rows
// go to the cache, else from it.
template <typename T, bool FP8, bool WRITE>
__global__ void __launch_bounds__(kThreads, WRITE ? 6 : 8) paged_copy_kernel(const CopyParams p) {
  constexpr int PIECE = kPiece<FP8>;
  constexpr int WORDS = PIECE / 8;  // 16-byte words of a packed piece
  __shared__ int s_page[kMaxTokens];            // < 0: the token has no place
  __shared__ int64_t s_row[2][kMaxTokens];      // its rows in K and V, of head 0
  __shared__ int64_t s_scale[2][kMaxTokens];
  let_next_launch();
  wait_for_launch_before();
  const int t0 = blockIdx.x * p.tokens;
  const int count = min(p.tokens, p.seqs.total - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lanes = 1 << p.lanes_log2;
  const int pieces = lanes * p.heads * 2;  // of a token
  const int n = pieces * count;

  // piece i of the run: its token, K or V, head, first element, and place in the packed rows
  struct Place {
    int tok, kv, head, elem;
  };
  auto place = [&](int i) -> Place {
    Place x;
    x.tok = static_cast<int>(__umulhi(static_cast<uint32_t>(i), p.pieces_inv));
    const int rest = i - x.tok * pieces;
    const int row = rest >> p.lanes_log2;
    x.kv = row >= p.heads;
    x.head = row - x.kv * p.heads;
    x.elem = (rest & (lanes - 1)) * PIECE;
    return x;
  };
  auto packed = [&](const Place& x) -> T* {
    return static_cast<T*>(p.rows[x.kv]) + static_cast<int64_t>(t0 + x.tok) * p.row_stride[x.kv][0] +
           x.head * p.row_stride[x.kv][1] + x.elem;
  };
  auto cached = [&](const Place& x) -> int64_t {
    return s_row[x.kv][x.tok] + x.head * p.cache_stride[x.kv][1] + x.elem;
  };
  auto scale_of = [&](const Place& x) -> float* {
    return p.scale[x.kv] + s_scale[x.kv][x.tok] + x.head * p.scale_stride[x.kv][1];
  };
  auto look_up = [&]() {
    for (int i = warp; i < count; i += kThreads / 32) {
      const int t = t0 + i;
      const int b = find_seq(p.seqs, t, lane);
      if (lane < 2) {  // K, V
        const int end = fresh(p.seqs.offsets + b + 1);
        int page = -2, pos = 0;  // -2: of no sequence
        if (t < end && t >= fresh(p.seqs.offsets + b)) {
          pos = fresh(p.seqs.kv_lens + b) - (end - t);
          page = page_of(p.seqs, b, pos);
          if (page < 0) report(p.seqs.status, kStatusPageTable);
        }
        const int slot = pos & ((1 << p.seqs.page_log2) - 1);
        if (lane == 0) s_page[i] = page;
        s_row[lane][i] = page * p.cache_stride[lane][0] + slot * p.cache_stride[lane][2];
        s_scale[lane][i] = page * p.scale_stride[lane][0] + slot;
      }
    }
    __syncthreads();
  };

  if (!WRITE) look_up();
  // every thread makes the same number of turns: the shuffles below take whole warps
  for (int at = 0; at < n; at += kThreads * kUnroll) {
    uint4 x[kUnroll][WORDS];
    float sc[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = at + u * kThreads + threadIdx.x;
      sc[u] = 0.f;
#pragma unroll
      for (int k = 0; k < WORDS; ++k) x[u][k] = make_uint4(0, 0, 0, 0);
      if (i < n) {
        const Place q = place(i);
        if (WRITE) {
#pragma unroll
          for (int k = 0; k < WORDS; ++k) x[u][k] = fresh(reinterpret_cast<const uint4*>(packed(q)) + k);
        } else if (s_page[q.tok] >= 0) {
          const int64_t c = cached(q);
          if (FP8) {
            x[u][0] = fresh(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.cache[q.kv]) + c));
            sc[u] = fresh(scale_of(q));
          } else {
            x[u][0] = fresh(reinterpret_cast<const uint4*>(static_cast<const T*>(p.cache[q.kv]) + c));
          }
        }
      }
    }
    if (WRITE && at == 0) look_up();
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = at + u * kThreads + threadIdx.x;
      const bool in = i < n;
      const Place q = place(in ? i : 0);
      const bool on = in && (WRITE ? s_page[q.tok] >= 0 : s_page[q.tok] != -2);
      if constexpr (!FP8) {
        if (on) *reinterpret_cast<uint4*>(WRITE ? static_cast<T*>(p.cache[q.kv]) + cached(q) : packed(q)) = x[u][0];
      } else if constexpr (WRITE) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = k < 4 ? (&x[u][0].x)[k] : (&x[u][WORDS - 1].x)[k - 4];
        // The row's largest magnitude: without their signs the bits of 16-bit floats are ordered as
        // their values are, two to a word.  What is not finite is rare: it becomes NaN and does not
        // count.  (Float by float this was half of the kernel's instructions, which bound it.)
        constexpr uint32_t kInf = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = __vmaxu2(m, w[k] & 0x7fff7fffu);
        if (__any_sync(0xffffffffu, (m & 0xffffu) >= kInf || m >> 16 >= kInf)) {
          m = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t keep = 0xffffffffu;
            if ((w[k] & 0x7fffu) >= kInf) keep &= 0xffff0000u;
            if ((w[k] >> 16 & 0x7fffu) >= kInf) keep &= 0x0000ffffu;
            m = __vmaxu2(m, w[k] & keep & 0x7fff7fffu);
            w[k] |= ~keep;
          }
        }
        for (int d = 1; d < lanes; d <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float top = Cvt16<T>::unpack(max(m & 0xffffu, m >> 16)).x;
        // top = (1 + man / 2^23) * 2^(ex - 127); 448 = 1.75 * 2^8.  (A subnormal top has ex = 0
        // and takes the smallest scale.)
        const uint32_t bits = __float_as_uint(top);
        int ex = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
        ex = top == 0.f ? 0 : max(ex, -126);
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        uint32_t c[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 a = fmul2(Cvt16<T>::unpack(w[2 * k]), make_float2(inv, inv));
          const float2 b = fmul2(Cvt16<T>::unpack(w[2 * k + 1]), make_float2(inv, inv));
          c[k] = pack2_e4m3(a.x, a.y) | (pack2_e4m3(b.x, b.y) << 16);
        }
        if (on) {
          *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.cache[q.kv]) + cached(q)) =
              make_uint4(c[0], c[1], c[2], c[3]);
          if (q.elem == 0) *scale_of(q) = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
        }
      } else {
        uint32_t out[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t w = (&x[u][0].x)[k >> 1];
          const uint32_t h2 = e4m3x2_to_h2(static_cast<uint16_t>(w >> (16 * (k & 1))));
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h2));
          const float2 y = fmul2(v, make_float2(sc[u], sc[u]));
          out[k] = pack2(y.x, y.y, static_cast<T*>(nullptr));
        }
        if (on) {
          uint4* dst = reinterpret_cast<uint4*>(packed(q));
          dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
          dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
        }
      }
    }
  }
}

int copy_rows(const FaPagedCopyArgs* a, void* stream, bool write) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(FaPagedCopyArgs)))
    return FA_ERR_INVALID_ARG;
  int rc = check_cache(a->cache, a->dtype, a->total);
  if (rc != FA_OK) return rc;
  if (a->total == 0 || a->cache.seqs == 0) return FA_OK;
  if (!a->k || !a->v) return FA_ERR_INVALID_ARG;
  CopyParams p{};
  p.rows[0] = a->k;
  p.rows[1] = a->v;
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = i ? a->v_stride : a->k_stride;
    if (reinterpret_cast<uintptr_t>(p.rows[i]) % 16 || (a->total > 1 && st[0] % 8) ||
        (a->cache.heads_kv > 1 && st[1] % 8))
      return FA_ERR_MISALIGNED;
    for (int d = 0; d < 2; ++d) p.row_stride[i][d] = st[d];
  }
  rc = check_device();
  if (rc != FA_OK) return rc;
  p.seqs = seqs_of(a->cache, a->total, a->dev_status);
  p.cache[0] = a->cache.k;
  p.cache[1] = a->cache.v;
  p.scale[0] = a->cache.k_scale;
  p.scale[1] = a->cache.v_scale;
  for (int d = 0; d < 3; ++d) {
    p.cache_stride[0][d] = a->cache.k_stride[d];
    p.cache_stride[1][d] = a->cache.v_stride[d];
  }
  for (int d = 0; d < 2; ++d) {
    p.scale_stride[0][d] = a->cache.k_scale_stride[d];
    p.scale_stride[1][d] = a->cache.v_scale_stride[d];
  }
  p.heads = static_cast<int>(a->cache.heads_kv);
  p.head_dim = static_cast<int>(a->cache.head_dim);
  // A CTA's run: enough tokens for one round of kUnroll pieces a thread, fewer where that would
  // leave SMs without a CTA.
  const bool f8 = a->cache.dtype == FA_DTYPE_FP8_E4M3, half = a->dtype == FA_DTYPE_FP16;
  const int64_t lanes = a->cache.head_dim / (f8 ? kPiece<true> : kPiece<false>);
  const int64_t pieces = lanes * a->cache.heads_kv * 2;
  int64_t tokens = kThreads * kUnroll / pieces;
  const int64_t share = a->total / (2 * sm_count_of_current());
  if (tokens > share) tokens = share;
  p.tokens = static_cast<int>(tokens < 1 ? 1 : tokens > kMaxTokens ? kMaxTokens : tokens);
  p.lanes_log2 = log2_of(lanes);
  p.pieces_inv = p.tokens == 1 ? 0u : static_cast<uint32_t>((int64_t{1} << 32) / pieces + 1);
  const int64_t grid = (a->total + p.tokens - 1) / p.tokens;
  const auto kernel = f8 && half ? (write ? paged_copy_kernel<__half, true, true>
                                          : paged_copy_kernel<__half, true, false>)
                      : f8       ? (write ? paged_copy_kernel<__nv_bfloat16, true, true>
                                          : paged_copy_kernel<__nv_bfloat16, true, false>)
                                 : (write ? paged_copy_kernel<__half, false, true>  // any 16 bits
                                          : paged_copy_kernel<__half, false, false>);
  return launch_dependent(kernel, dim3(static_cast<unsigned>(grid)), kThreads, 0,
                          static_cast<cudaStream_t>(stream), p);
}

}  // namespace
}  // namespace fa

extern "C" {

int fa_paged_write_sm100(const FaPagedCopyArgs* args, void* stream) {
  return fa::copy_rows(args, stream, true);
}

int fa_paged_read_sm100(const FaPagedCopyArgs* args, void* stream) {
  return fa::copy_rows(args, stream, false);
}

}  // extern "C"
