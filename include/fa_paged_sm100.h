/*
 * C ABI of the paged key/value cache of the B200 (sm_100a) attention: writing new tokens into it,
 * reading tokens back, and attention of ragged chunks of new tokens over it.
 *
 * The cache.  `k` and `v` are [num_pages, heads_kv, page_size, head_dim] with their own element
 * strides for (page, head, row); head_dim is contiguous.  fp16 and bf16 caches hold the values;
 * a float8 e4m3 cache (FA_DTYPE_FP8_E4M3) holds value / scale, with one fp32 scale per
 * (page, head, row) in `k_scale` and `v_scale` (the row dimension contiguous).
 *
 * The sequences.  `page_table` [seqs, table_cols] lists the pages of each sequence in order; the
 * entries behind a sequence's last page are not read.  `kv_lens` [seqs] is each sequence's length
 * in the cache, its new tokens included.  `offsets` [seqs + 1] gives its rows in the packed
 * tensors [total, heads, head_dim]: row i of sequence b is row offsets[b] + i there and the token
 * at position kv_lens[b] - (offsets[b + 1] - offsets[b]) + i of the sequence.  Packed rows of no
 * sequence (behind offsets[seqs], or before offsets[0]) are padding: outputs there are not written, and
 * what inputs hold there does not matter, but it may be read, so all `total` rows have to be there.  All
 * three are int32 device arrays.
 *
 * Lengths, offsets (which do not decrease) and pages are device data that must not change while a call
 * runs: a kernel reads them more than once.  They are checked by the kernels: what lies outside the table
 * or the cache is not accessed, FA_ERR_PAGE_TABLE is written to *dev_status, and the results of the
 * sequence concerned are undefined.
 *
 * Conventions as in fa_fwd_sm100.h: the caller owns every buffer, the library allocates no device
 * memory, launches are asynchronous on `stream`, errors seen on the host come back before
 * anything is enqueued.
 */
#ifndef FA_PAGED_SM100_H_
#define FA_PAGED_SM100_H_

#include <stdint.h>

#include "fa_fwd_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache element type besides FaDtype's fp16 and bf16. */
enum FaCacheDtype { FA_DTYPE_FP8_E4M3 = 3 };

typedef struct FaPagedCache {
  void* k;
  void* v;
  float* k_scale; /* float8 caches only, else NULL */
  float* v_scale;
  const int32_t* page_table;
  const int32_t* offsets;
  const int32_t* kv_lens;
  int64_t k_stride[3]; /* element strides of (page, head, row) */
  int64_t v_stride[3];
  int64_t k_scale_stride[2]; /* element strides of (page, head); rows are contiguous */
  int64_t v_scale_stride[2];
  int64_t num_pages;
  int64_t heads_kv;
  int64_t page_size; /* tokens per page: a power of two, 8 .. 1024 */
  int64_t head_dim;  /* 16, 32, 64, 128 or 256 */
  int64_t table_stride; /* elements between the rows of page_table */
  int64_t table_cols;
  int64_t seqs;
  int32_t dtype; /* FA_DTYPE_FP16, FA_DTYPE_BF16 or FA_DTYPE_FP8_E4M3 */
} FaPagedCache;

/* Packed rows [total, heads_kv, head_dim] of keys and values, to or from the cache. */
typedef struct FaPagedCopyArgs {
  int32_t struct_size; /* sizeof(FaPagedCopyArgs) */
  void* k;
  void* v;
  int32_t* dev_status; /* optional device int, 0 on success */
  FaPagedCache cache;
  int64_t k_stride[2]; /* element strides of (row, head); multiples of 16 bytes */
  int64_t v_stride[2];
  int64_t total;
  int32_t dtype; /* FA_DTYPE_FP16 or FA_DTYPE_BF16; the cache's own unless that is float8 */
} FaPagedCopyArgs;

typedef struct FaPagedAttnArgs {
  int32_t struct_size; /* sizeof(FaPagedAttnArgs) */
  const void* q; /* [total, heads_q, head_dim] */
  void* o;
  float* lse;          /* [total, heads_q], contiguous */
  void* workspace;     /* fa_paged_workspace_bytes() bytes, 256-byte aligned; needs no clearing */
  int32_t* dev_status; /* optional device int, 0 on success */
  FaPagedCache cache;
  int64_t q_stride[2]; /* element strides of (row, head); multiples of 16 bytes */
  int64_t o_stride[2];
  int64_t total;
  int64_t heads_q;   /* a multiple of heads_kv */
  int64_t max_q_len; /* upper bound of a sequence's new tokens that the kernel choice goes by
                        (0: total); a longer sequence is computed all the same */
  int64_t workspace_bytes;
  int32_t dtype;  /* of q and o: the cache's own, or fp16 / bf16 with a float8 cache */
  int32_t causal; /* a token attends to positions up to its own; 0: to the whole sequence */
  float sm_scale;
} FaPagedAttnArgs;

/* Write the packed rows into the cache.  Rows of a float8 cache are stored as
 * round_e4m3(x / s), s = 2^e with the smallest e >= -126 for which the largest finite |x| of the
 * row is at most 448 s (s = 1 for a row of zeros); infinities and NaN are stored as NaN. */
FA_API int fa_paged_write_sm100(const FaPagedCopyArgs* args, void* stream);

/* Read packed rows from the cache, dequantised and rounded once. */
FA_API int fa_paged_read_sm100(const FaPagedCopyArgs* args, void* stream);

/* Attention of the packed queries over the cache: out, and the natural-log logsumexp.  A row
 * with no key to attend to gets out = 0 and lse = -inf.  Every value inside a sequence takes part, with
 * a probability of 0 where the causal mask hides it, so a NaN or an infinity among them may show in any
 * row of the sequence.  Over a float8 cache, calls of more than 32 query rows (new tokens times
 * heads_q / heads_kv; max_q_len counts) round code * scale to q's type.  That is exact for scales that
 * fa_paged_write_sm100 left for rows of q's type, up to 63488 in fp16 (which e4m3 does not round up to
 * 65536); otherwise it is a rounding more, and with fp16 queries what lies beyond 65504 becomes infinite.
 * Scales: positive, normal numbers; up to 32 query rows, values 2^-80 below the largest that a row's
 * sequence holds may be left out of account. */
FA_API int fa_paged_attn_sm100(const FaPagedAttnArgs* args, void* stream);

/* Workspace of fa_paged_attn_sm100 for these arguments (pointers are not looked at), on the
 * current device; negative: a FaStatus. */
FA_API int64_t fa_paged_workspace_bytes(const FaPagedAttnArgs* args);

#ifdef __cplusplus
}
#endif

#endif /* FA_PAGED_SM100_H_ */
