// C-ABI front end of the sm_100a FlashAttention forward (declared in include/fa_fwd_sm100.h).
//
// Host-side duties, in the order the reference's launcher performs them
// (`_launch_kernel`, flash_attention_forward.py:1130-1194):
//   validate shapes / head_dim (reference `_validate_inputs`, :1114-1122)
//   resolve the tile config (reference `_resolve_tiling`, :626-631)
//   size the grid (reference `_build_grid`, :1125-1127)
//   launch on the caller's stream (reference `_attn_fwd[grid](...)`, :1159-1193)
// plus what TMA needs: one CUtensorMap per tensor, encoded through the driver entry point
// obtained from the runtime (no link against libcuda).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <mutex>

#include "../../include/fa_fwd_sm100.h"
#include "../../include/fa_paged_sm100.h"
#include "fa_fp32.h"
#include "fa_launch.h"

namespace {

constexpr int kSmemLimit = 232448;  // 227 KiB opt-in dynamic shared memory per block (sm_100)
constexpr int kMaxStagesAllowed = 8;

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Per-device "is this an sm_100 part" cache (16 devices is plenty for one node).
int device_ok(int dev) {
  static std::atomic<int> cache[16] = {};  // 0 unknown, 1 ok, -1 not ok
  if (dev < 0 || dev >= 16) return 0;
  int known = cache[dev].load(std::memory_order_relaxed);
  if (known == 0) {
    int major = 0, minor = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess) {
      (void)cudaGetLastError();
      return 0;
    }
    known = (major == 10 && minor == 0) ? 1 : -1;
    cache[dev].store(known, std::memory_order_relaxed);
  }
  return known == 1;
}

// Streaming multiprocessors of a device (cached; 148 on B200).
int sm_count(int dev) {
  static std::atomic<int> cache[16] = {};
  if (dev < 0 || dev >= 16) return 148;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = 148;
    }
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Element type of a tensor map: an FaDtype, or one byte (fp8 V).
constexpr int kDtypeByte = 100;

int elt_bytes(int dtype) {
  return dtype == FA_DTYPE_FP32 ? 4 : (dtype == kDtypeByte ? 1 : 2);
}

bool v_fp8(const FaFwdArgs* a) { return (a->flags & FA_FLAG_V_FP8_E5M2) != 0; }

bool head_dim_ok(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128 || d == 256; }

fa::KernelInfo info_for(int64_t head_dim, int dtype, int block_n, int qt, bool vf8 = false) {
  switch (head_dim) {
    case 16: return fa::info_d16(dtype, block_n, qt, vf8);
    case 32: return fa::info_d32(dtype, block_n, qt, vf8);
    case 64: return fa::info_d64(dtype, block_n, qt, vf8);
    case 128: return fa::info_d128(dtype, block_n, qt, vf8);
    case 256: return fa::info_d256(dtype, block_n, qt, vf8);
    default: return fa::KernelInfo{false, 0, 0, 0, 0, 0, 0, 0, 0};
  }
}

int max_stages_for(const fa::KernelInfo& ki) {
  if (!ki.exists) return 0;
  const int s = (kSmemLimit - ki.smem_fixed) / ki.kv_tile_bytes;
  return std::min(s, kMaxStagesAllowed);
}

// The persistent warp-specialised kernel (fa_fwd_ws.cuh) serves fp16 / bf16 at head_dim 64 and
// 128 with (block_m, block_n) = (256, 128); every other configuration runs one CTA per tile.
bool ws_shape(int64_t head_dim, int dtype, int block_m, int block_n) {
  return (dtype == FA_DTYPE_FP16 || dtype == FA_DTYPE_BF16) && (head_dim == 64 || head_dim == 128) &&
         block_m == 256 && block_n == 128;
}

int ws_max_stages(int64_t head_dim) {
  const int fixed = head_dim == 64 ? fa::ws_smem_fixed<64>() : fa::ws_smem_fixed<128>();
  const int stage = head_dim == 64 ? fa::ws_stage_bytes<64>() : fa::ws_stage_bytes<128>();
  return std::min((kSmemLimit - fixed) / stage, kMaxStagesAllowed);
}

// Ring depth limit of the kernel that serves these knobs (0 if none).  For the shapes both
// kernels serve this is the smaller (persistent) limit, so a ring depth is valid whichever
// of the two a call dispatches to.
int stage_limit(int64_t head_dim, int dtype, int block_m, int block_n, bool vf8) {
  if (!vf8 && ws_shape(head_dim, dtype, block_m, block_n)) return ws_max_stages(head_dim);
  return max_stages_for(info_for(head_dim, dtype, block_n, block_m / 128, vf8));
}

// Encode a 4-D tiled map over a [B, H, S, D] tensor with dims listed innermost first.
int encode_map(CUtensorMap* map, const void* ptr, int dtype, int64_t B, int64_t H, int64_t S,
               int64_t D, const int64_t st[3], int box_cols, int box_rows, int swz_bytes,
               bool atom32 = false) {
  const int eb = elt_bytes(dtype);
  if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return FA_ERR_MISALIGNED;
  // element strides -> byte strides for (seq, head, batch); size-1 dims get a harmless value
  int64_t s_seq = st[2] * eb, s_head = st[1] * eb, s_batch = st[0] * eb;
  if (S == 1) s_seq = ((D * eb + 15) / 16) * 16;
  if (H == 1) s_head = s_seq * S;
  if (B == 1) s_batch = s_head * H;
  for (int64_t s : {s_seq, s_head, s_batch})
    if (s <= 0 || s % 16 != 0 || s >= (int64_t{1} << 40)) return FA_ERR_MISALIGNED;
  auto enc = encode_fn();
  if (!enc) return FA_ERR_TENSOR_MAP;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S),
                              static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(s_seq), static_cast<cuuint64_t>(s_head),
                                 static_cast<cuuint64_t>(s_batch)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows),
                             1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  CUtensorMapDataType dt = dtype == FA_DTYPE_FP16   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                           : dtype == FA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                           : dtype == kDtypeByte    ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  CUtensorMapSwizzle sw = atom32             ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B
                          : swz_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                          : swz_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                          : swz_bytes == 32 ? CU_TENSOR_MAP_SWIZZLE_32B
                                            : CU_TENSOR_MAP_SWIZZLE_NONE;
  CUresult r = enc(map, dt, 4, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FA_OK : FA_ERR_TENSOR_MAP;
}

int validate(const FaFwdArgs* a) {
  if (!a || a->struct_size != static_cast<int32_t>(sizeof(FaFwdArgs))) return FA_ERR_INVALID_ARG;
  if (a->batch <= 0 || a->heads <= 0 || a->seqlen <= 0) return FA_ERR_INVALID_ARG;
  if (a->seqlen > (int64_t{1} << 30) || a->batch * a->heads > (int64_t{1} << 30))
    return FA_ERR_INVALID_ARG;
  if (!head_dim_ok(a->head_dim)) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  if (a->dtype != FA_DTYPE_FP16 && a->dtype != FA_DTYPE_BF16 && a->dtype != FA_DTYPE_FP32)
    return FA_ERR_UNSUPPORTED_DTYPE;
  if (!a->q || !a->k || !a->v || !a->o || !a->lse) return FA_ERR_INVALID_ARG;
  if (!std::isfinite(a->sm_scale)) return FA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(a->lse) % 4 != 0) return FA_ERR_MISALIGNED;
  if (a->flags & ~(FA_FLAG_FP32_TF32 | FA_FLAG_V_FP8_E5M2 | FA_FLAG_ONE_CTA_PER_TILE))
    return FA_ERR_INVALID_ARG;
  if (v_fp8(a)) {
    if (a->dtype == FA_DTYPE_FP32) return FA_ERR_UNSUPPORTED_DTYPE;
    if (a->head_dim < 32) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  }
  return FA_OK;
}

// fp32 inputs without FA_FLAG_FP32_TF32 take the CUDA-core kernel.
bool use_fp32_simt(const FaFwdArgs* a) {
  return a->dtype == FA_DTYPE_FP32 && !(a->flags & FA_FLAG_FP32_TF32);
}

// True when this call runs on the persistent kernel: every shape it serves (fp16 / bf16,
// head_dim 64 / 128, 256 x 128 tile) with a positive scale, unless the caller asks for one CTA
// per tile.  Measured on B200 against the one-CTA-per-tile kernel: causal shapes +5..+12 %,
// outlier-heavy rows +20..+30 %, long non-causal N(0, 1) inputs within +-2 %.
bool use_ws(const FaFwdArgs* a, const FaTileConfig& t) {
  return !v_fp8(a) && !(a->flags & FA_FLAG_ONE_CTA_PER_TILE) && a->sm_scale > 0.f &&
         ws_shape(a->head_dim, a->dtype, t.block_m, t.block_n);
}

int resolve_tile(const FaFwdArgs* a, FaTileConfig* t) {
  *t = a->tile;
  if (t->block_m == 0 && t->block_n == 0) {
    int rc = fa_fwd_sm100_default_tile(a->head_dim, a->dtype, a->causal, a->seqlen, t);
    if (rc != FA_OK) return rc;
    t->num_stages = a->tile.num_stages;
    t->persistent_ctas = a->tile.persistent_ctas;
  }
  if (t->block_m != 128 && t->block_m != 256) return FA_ERR_UNSUPPORTED_TILE;
  if (t->block_n != 64 && t->block_n != 128) return FA_ERR_UNSUPPORTED_TILE;
  const fa::KernelInfo ki = info_for(a->head_dim, a->dtype, t->block_n, t->block_m / 128, v_fp8(a));
  if (!ki.exists) return FA_ERR_UNSUPPORTED_TILE;
  const int smax = stage_limit(a->head_dim, a->dtype, t->block_m, t->block_n, v_fp8(a));
  if (smax < 2) return FA_ERR_UNSUPPORTED_TILE;
  if (t->num_stages == 0) t->num_stages = smax;
  if (t->num_stages < 2 || t->num_stages > smax) return FA_ERR_UNSUPPORTED_TILE;
  if (t->persistent_ctas < 0) return FA_ERR_UNSUPPORTED_TILE;
  // A persistent grid size only means something to the persistent kernel: refuse it elsewhere
  // rather than accept a setting that would not be applied.
  if (t->persistent_ctas > 0 && !use_ws(a, *t)) return FA_ERR_UNSUPPORTED_TILE;
  return FA_OK;
}

}  // namespace

namespace fa {
int check_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return FA_ERR_DEVICE;
  }
  return device_ok(dev) ? FA_OK : FA_ERR_DEVICE;
}

int sm_count_of_current() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    dev = -1;
  }
  return sm_count(dev);
}

int encode_cache_map(CUtensorMap* map, const void* ptr, int dtype, int64_t pages, int64_t heads,
                     int64_t rows, int64_t head_dim, const int64_t st[3], int box_cols,
                     int box_rows, int swz_bytes) {
  return encode_map(map, ptr, dtype == FA_DTYPE_FP8_E4M3 ? kDtypeByte : dtype, pages, heads, rows,
                    head_dim, st, box_cols, box_rows, swz_bytes);
}

int encode_query_map(CUtensorMap* map, const void* ptr, int dtype, int64_t total, int64_t heads,
                     int64_t head_dim, const int64_t st[2], int box_cols, int box_heads,
                     int box_tokens, int swz_bytes) {
  const int64_t s_head = st[1] * 2, s_tok = st[0] * 2;
  if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return FA_ERR_MISALIGNED;
  for (int64_t s : {s_head, s_tok})
    if (s <= 0 || s % 16 != 0 || s >= (int64_t{1} << 40)) return FA_ERR_MISALIGNED;
  auto enc = encode_fn();
  if (!enc) return FA_ERR_TENSOR_MAP;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(total)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(s_head), static_cast<cuuint64_t>(s_tok)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_heads),
                             static_cast<cuuint32_t>(box_tokens)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      enc(map, dtype == FA_DTYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
          3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
          swz_bytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
          : swz_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                            : CU_TENSOR_MAP_SWIZZLE_32B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FA_OK : FA_ERR_TENSOR_MAP;
}

KernelInfo kernel_info(int head_dim, int dtype, int block_n, int qt, bool vf8) {
  return info_for(head_dim, dtype, block_n, qt, vf8);
}
}  // namespace fa

extern "C" {

int fa_fwd_sm100_default_tile(int64_t head_dim, int32_t dtype, int32_t causal, int64_t seqlen,
                              FaTileConfig* cfg) {
  (void)causal;
  if (!cfg) return FA_ERR_INVALID_ARG;
  if (!head_dim_ok(head_dim)) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  if (dtype != FA_DTYPE_FP16 && dtype != FA_DTYPE_BF16 && dtype != FA_DTYPE_FP32)
    return FA_ERR_UNSUPPORTED_DTYPE;
  FaTileConfig t{};
  if (dtype == FA_DTYPE_FP32) {
    if (head_dim > 128 || head_dim < 32) return FA_ERR_UNSUPPORTED_TILE;
    t.block_m = 128;
    t.block_n = 64;
  } else if (head_dim == 256) {
    t.block_m = 128;
    t.block_n = 64;
  } else {
    // Two 128-row query tiles share every K/V tile; a single tile for short sequences.
    t.block_m = seqlen > 128 ? 256 : 128;
    t.block_n = 128;
  }
  t.num_stages = 0;
  t.persistent_ctas = 0;
  *cfg = t;
  return FA_OK;
}

int fa_fwd_sm100_supported(int64_t head_dim, int32_t dtype, int32_t block_m, int32_t block_n,
                           int32_t num_stages) {
  if (!head_dim_ok(head_dim)) return 0;
  if (block_m != 128 && block_m != 256) return 0;
  if (block_n != 64 && block_n != 128) return 0;
  if (!info_for(head_dim, dtype, block_n, block_m / 128).exists) return 0;
  const int smax = stage_limit(head_dim, dtype, block_m, block_n, false);
  if (smax < 2) return 0;
  if (num_stages == 0) return 1;
  return (num_stages >= 2 && num_stages <= smax) ? 1 : 0;
}

int fa_fwd_sm100_max_stages(int64_t head_dim, int32_t dtype, int32_t block_m, int32_t block_n) {
  if (!head_dim_ok(head_dim) || (block_m != 128 && block_m != 256)) return 0;
  if (block_n != 64 && block_n != 128) return 0;
  if (!info_for(head_dim, dtype, block_n, block_m / 128).exists) return 0;
  const int s = stage_limit(head_dim, dtype, block_m, block_n, false);
  return s >= 2 ? s : 0;
}

int64_t fa_fwd_sm100_grid_size(const FaFwdArgs* a) {
  if (validate(a) != FA_OK) return -1;
  if (use_fp32_simt(a)) return ((a->seqlen + 63) / 64) * a->batch * a->heads;
  FaTileConfig t;
  if (resolve_tile(a, &t) != FA_OK) return -1;
  const int64_t nq = (a->seqlen + t.block_m - 1) / t.block_m;
  const int64_t tiles = nq * a->batch * a->heads;
  if (!use_ws(a, t)) return tiles;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    dev = -1;
  }
  const int64_t ctas = t.persistent_ctas > 0 ? t.persistent_ctas : sm_count(dev);
  return std::min(tiles, ctas);
}

int fa_fwd_sm100(const FaFwdArgs* a, void* stream) {
  int rc = validate(a);
  if (rc != FA_OK) return rc;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return FA_ERR_DEVICE;
  }
  if (!device_ok(dev)) return FA_ERR_DEVICE;
  if (use_fp32_simt(a)) {
    fa::Fp32Params fp{};
    fp.batch = a->batch;
    fp.heads = a->heads;
    fp.seqlen = static_cast<int>(a->seqlen);
    fp.head_dim = static_cast<int>(a->head_dim);
    for (int i = 0; i < 3; ++i) {
      fp.q_stride[i] = a->q_stride[i];
      fp.k_stride[i] = a->k_stride[i];
      fp.v_stride[i] = a->v_stride[i];
      fp.o_stride[i] = a->o_stride[i];
    }
    fp.causal = a->causal ? 1 : 0;
    fp.scale_log2 = a->sm_scale * fa::kLog2e;
    return fa::launch_fp32_simt(static_cast<const float*>(a->q), static_cast<const float*>(a->k),
                                static_cast<const float*>(a->v), static_cast<float*>(a->o),
                                a->lse, fp, static_cast<cudaStream_t>(stream));
  }
  FaTileConfig t;
  rc = resolve_tile(a, &t);
  if (rc != FA_OK) return rc;
  const int qt = t.block_m / 128;
  const bool vf8 = v_fp8(a);
  const fa::KernelInfo ki = info_for(a->head_dim, a->dtype, t.block_n, qt, vf8);

  fa::LaunchPlan lp;
  std::memset(&lp, 0, sizeof(lp));
  const int64_t B = a->batch, H = a->heads, S = a->seqlen, D = a->head_dim;
  rc = encode_map(&lp.tmQ, a->q, a->dtype, B, H, S, D, a->q_stride, ki.box_cols, 128, ki.swz_bytes);
  if (rc == FA_OK)
    rc = encode_map(&lp.tmK, a->k, a->dtype, B, H, S, D, a->k_stride, ki.box_cols, t.block_n,
                    ki.swz_bytes);
  if (rc == FA_OK)
    rc = encode_map(&lp.tmV, a->v, vf8 ? kDtypeByte : a->dtype, B, H, S, D, a->v_stride,
                    ki.v_box_cols, t.block_n, ki.v_swz_bytes, /*atom32=*/a->dtype == FA_DTYPE_FP32);
  // The persistent kernel stores O in 128 x 32 boxes with a 64-byte swizzle.
  const bool ws = use_ws(a, t);
  if (rc == FA_OK)
    rc = ws ? encode_map(&lp.tmO, a->o, a->dtype, B, H, S, D, a->o_stride, 32, 128, 64)
            : encode_map(&lp.tmO, a->o, a->dtype, B, H, S, D, a->o_stride, ki.box_cols, 128,
                         ki.swz_bytes);
  if (rc != FA_OK) return rc;

  const int64_t nq = (S + t.block_m - 1) / t.block_m;
  lp.grid = nq * B * H;
  if (lp.grid > 0x7fffffffLL) return FA_ERR_INVALID_ARG;
  lp.ws = ws;
  if (lp.ws) {
    fa::WsParams& w = lp.ws_params;
    w.batch = static_cast<int>(B);
    w.heads = static_cast<int>(H);
    w.seqlen = static_cast<int>(S);
    w.n_qblocks = static_cast<int>(nq);
    w.total_tiles = static_cast<int>(lp.grid);
    w.causal = a->causal ? 1 : 0;
    w.stages = t.num_stages;
    w.scale_log2 = a->sm_scale * fa::kLog2e;
    w.lse = a->lse;
    w.status = a->dev_status;
    const int64_t ctas = t.persistent_ctas > 0 ? t.persistent_ctas : sm_count(dev);
    lp.grid = std::min<int64_t>(lp.grid, ctas);
  }
  lp.params.batch = static_cast<int>(B);
  lp.params.heads = static_cast<int>(H);
  lp.params.seqlen = static_cast<int>(S);
  lp.params.n_qblocks = static_cast<int>(nq);
  lp.params.causal = a->causal ? 1 : 0;
  lp.params.stages = t.num_stages;
  lp.params.scale_log2 = a->sm_scale * fa::kLog2e;
  lp.params.lse = a->lse;
  lp.params.status = a->dev_status;
  lp.dtype = a->dtype;
  lp.block_n = t.block_n;
  lp.qt = qt;
  lp.vf8 = vf8;
  lp.stream = static_cast<cudaStream_t>(stream);

  switch (D) {
    case 16: return fa::launch_d16(lp);
    case 32: return fa::launch_d32(lp);
    case 64: return fa::launch_d64(lp);
    case 128: return fa::launch_d128(lp);
    case 256: return fa::launch_d256(lp);
    default: return FA_ERR_UNSUPPORTED_HEAD_DIM;
  }
}

const char* fa_fwd_sm100_status_string(int code) {
  switch (code) {
    case FA_OK: return "ok";
    case FA_ERR_INVALID_ARG: return "invalid argument";
    case FA_ERR_UNSUPPORTED_HEAD_DIM: return "HEAD_DIM must be one of {16, 32, 64, 128, 256}";
    case FA_ERR_UNSUPPORTED_DTYPE: return "dtype must be float16, bfloat16 or float32";
    case FA_ERR_MISALIGNED:
      return "tensor pointer or stride is not 16-byte aligned (TMA requirement)";
    case FA_ERR_UNSUPPORTED_TILE: return "tile configuration not available for this head_dim/dtype";
    case FA_ERR_TENSOR_MAP: return "cuTensorMapEncodeTiled failed";
    case FA_ERR_LAUNCH: return "kernel launch failed";
    case FA_ERR_DEVICE: return "current CUDA device is not an sm_100 (B200) part";
    case FA_ERR_DEVICE_TIMEOUT: return "a pipeline wait in the kernel timed out";
    case FA_ERR_PAGE_TABLE:
      return "a page index, length or offset of a paged call lies outside its page table or cache";
    default: return "unknown status";
  }
}

int fa_fwd_sm100_version(void) { return 1000; }

}  // extern "C"
