// Writing packed rows of new tokens into the paged key/value cache, and reading rows back
// (declared in include/fa_paged_sm100.h).
//
// A row is one (token, kv head) of K or V: head_dim values.  Float8 rows are quantised by
//   s = 2^e, e = min{ e >= -126 : max |x| <= 448 * 2^e },   c = round_e4m3(x / s).
// A power of two costs e4m3 nothing (a floating-point format keeps its relative step at any
// magnitude; only rows that spread over more than 2^14 reach its subnormals), makes x / s, c * s
// and the scale itself exact, and leaves the one rounding to 4 bits.
//
// Both directions are bound by memory: each value is read and written once, in 16-byte pieces
// (8 values, 8 bytes on the float8 side), head_dim / 8 threads to a row, so that a row's largest
// magnitude is a few shuffles.  Each CTA takes a run of tokens: its warps first look up the
// sequence and the page of one token each (a 32-way search of the offsets), then all threads move
// the run's rows, kUnroll pieces in flight each.
#include <cmath>

#include "../../include/fa_paged_sm100.h"
#include "fa_paged_host.h"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 64;  // tokens of one CTA's run
constexpr int kUnroll = 4;

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
  int tokens;  // per CTA
};

// Smallest b with offsets[b + 1] > t, by the whole warp (seqs - 1 if there is none).
__device__ __forceinline__ int find_seq(const PagedSeqs& s, int t, int lane) {
  int lo = 0, hi = s.seqs - 1;  // the answer lies in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int probe = min(lo + (lane + 1) * step, hi);  // is the answer >= probe?
    const bool past = __ldg(s.offsets + probe) <= t;
    const int n = __popc(__ballot_sync(0xffffffffu, past));
    const int next = min(lo + n * step, hi);
    hi = n == 32 ? hi : min(lo + (n + 1) * step, hi) - 1;
    lo = next;
    hi = max(hi, lo);
  }
  return lo;
}

// T: type of the packed rows.  FP8: the cache holds e4m3 codes and scales, else T.  WRITE: rows
// go to the cache, else from it.
template <typename T, bool FP8, bool WRITE>
__global__ void __launch_bounds__(kThreads) paged_copy_kernel(const CopyParams p) {
  __shared__ int s_page[kMaxTokens];
  __shared__ int s_slot[kMaxTokens];
  const int t0 = blockIdx.x * p.tokens;
  const int count = min(p.tokens, p.seqs.total - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < count; i += kThreads / 32) {
    const int t = t0 + i;
    const int b = find_seq(p.seqs, t, lane);
    if (lane == 0) {
      const int end = __ldg(p.seqs.offsets + b + 1);
      int page = -2, pos = 0;  // -2: behind the last sequence
      if (t < end && t >= __ldg(p.seqs.offsets + b)) {
        pos = __ldg(p.seqs.kv_lens + b) - (end - t);
        page = page_of(p.seqs, b, pos);
        if (page < 0) report(p.seqs.status, kStatusPageTable);
      }
      s_page[i] = page;
      s_slot[i] = pos & ((1 << p.seqs.page_log2) - 1);
    }
  }
  __syncthreads();

  const int lanes = p.head_dim >> 3;            // threads of a row: 2 .. 32
  const int pieces = lanes * p.heads * 2;       // of a token
  const int n = pieces * count;
  // every thread makes the same number of turns: the shuffles below take whole warps
  for (int at = 0; at < n; at += kThreads * kUnroll) {
    uint4 x[kUnroll];
    float sc[kUnroll];
    int64_t packed[kUnroll], held[kUnroll], held_scale[kUnroll];
    int kv[kUnroll];
    bool on[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = at + u * kThreads + threadIdx.x;
      on[u] = i < n;
      const int tok = on[u] ? i / pieces : 0;
      const int rest = i - tok * pieces;
      const int piece = rest & (lanes - 1);
      const int hv = rest / lanes;
      kv[u] = hv >= p.heads;
      const int h = hv - kv[u] * p.heads;
      const int page = s_page[tok];
      on[u] = on[u] && page != -2 && (!WRITE || page >= 0);
      packed[u] = (t0 + tok) * p.row_stride[kv[u]][0] + h * p.row_stride[kv[u]][1] + piece * 8;
      const int64_t pg = page;
      held[u] = pg < 0 ? -1
                       : pg * p.cache_stride[kv[u]][0] + h * p.cache_stride[kv[u]][1] +
                             s_slot[tok] * p.cache_stride[kv[u]][2] + piece * 8;
      if (FP8)
        held_scale[u] = pg * p.scale_stride[kv[u]][0] + h * p.scale_stride[kv[u]][1] + s_slot[tok];
      x[u] = make_uint4(0, 0, 0, 0);
      sc[u] = 0.f;
      if (WRITE) {
        if (on[u])
          x[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.rows[kv[u]]) +
                                                      packed[u]));
      } else if (on[u] && held[u] >= 0) {
        if (FP8) {
          const uint2 c = __ldg(reinterpret_cast<const uint2*>(
              static_cast<const uint8_t*>(p.cache[kv[u]]) + held[u]));
          x[u].x = c.x;
          x[u].y = c.y;
          sc[u] = __ldg(p.scale[kv[u]] + held_scale[u]);
        } else {
          x[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.cache[kv[u]]) +
                                                      held[u]));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!FP8) {
        T* dst = WRITE ? static_cast<T*>(p.cache[kv[u]]) + held[u]
                       : static_cast<T*>(p.rows[kv[u]]) + packed[u];
        if (on[u]) *reinterpret_cast<uint4*>(dst) = x[u];
      } else if (WRITE) {
        float2 f[4] = {Cvt16<T>::unpack(x[u].x), Cvt16<T>::unpack(x[u].y),
                       Cvt16<T>::unpack(x[u].z), Cvt16<T>::unpack(x[u].w)};
        float top = 0.f;
        float* e = reinterpret_cast<float*>(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float a = fabsf(e[k]);
          if (a < INFINITY) top = fmaxf(top, a);
          else e[k] = NAN;
        }
        for (int d = 1; d < lanes; d <<= 1)
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // top = (1 + man / 2^23) * 2^(ex - 127); 448 = 1.75 * 2^8.  (A subnormal top has ex = 0
        // and takes the smallest scale.)
        const uint32_t bits = __float_as_uint(top);
        int ex = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
        ex = top == 0.f ? 0 : max(ex, -126);
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
        uint2 c;
        c.x = pack2_e4m3(e[0] * inv, e[1] * inv) | (pack2_e4m3(e[2] * inv, e[3] * inv) << 16);
        c.y = pack2_e4m3(e[4] * inv, e[5] * inv) | (pack2_e4m3(e[6] * inv, e[7] * inv) << 16);
        if (on[u]) {
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.cache[kv[u]]) + held[u]) = c;
          if ((threadIdx.x & (lanes - 1)) == 0)
            p.scale[kv[u]][held_scale[u]] = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
        }
      } else {
        uint32_t out[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w = k < 2 ? x[u].x : x[u].y;
          const uint32_t h2 = e4m3x2_to_h2(static_cast<uint16_t>(w >> (16 * (k & 1))));
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h2));
          if constexpr (sizeof(T) == 2) {
            const T a = static_cast<T>(v.x * sc[u]), z = static_cast<T>(v.y * sc[u]);
            out[k] = *reinterpret_cast<const uint16_t*>(&a) |
                     (static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&z)) << 16);
          }
        }
        if (on[u])
          *reinterpret_cast<uint4*>(static_cast<T*>(p.rows[kv[u]]) + packed[u]) =
              make_uint4(out[0], out[1], out[2], out[3]);
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
  // A CTA's run: enough tokens for two rounds of kUnroll pieces a thread, fewer where that would
  // leave SMs without a CTA.
  const int64_t pieces = a->cache.head_dim / 8 * a->cache.heads_kv * 2;
  int64_t tokens = 2 * kThreads * kUnroll / pieces;
  const int64_t share = a->total / (4 * sm_count_of_current());
  if (tokens > share) tokens = share;
  p.tokens = static_cast<int>(tokens < 1 ? 1 : tokens > kMaxTokens ? kMaxTokens : tokens);
  const int64_t grid = (a->total + p.tokens - 1) / p.tokens;
  const dim3 g(static_cast<unsigned>(grid)), t(kThreads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f8 = a->cache.dtype == FA_DTYPE_FP8_E4M3, half = a->dtype == FA_DTYPE_FP16;
  if (f8 && half && write) paged_copy_kernel<__half, true, true><<<g, t, 0, st>>>(p);
  else if (f8 && half) paged_copy_kernel<__half, true, false><<<g, t, 0, st>>>(p);
  else if (f8 && write) paged_copy_kernel<__nv_bfloat16, true, true><<<g, t, 0, st>>>(p);
  else if (f8) paged_copy_kernel<__nv_bfloat16, true, false><<<g, t, 0, st>>>(p);
  else if (write) paged_copy_kernel<__half, false, true><<<g, t, 0, st>>>(p);  // any 16-bit type
  else paged_copy_kernel<__half, false, false><<<g, t, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
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
