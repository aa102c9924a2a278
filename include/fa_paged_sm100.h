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

/* Attention behind shared prefixes: a row attends to a prefix that its group shares, and to its own
 * sequence behind that.  Prefix g is `prefix_lens[g]` tokens in the pages `prefix_table[g]` of the same
 * cache, and its group the packed rows prefix_offsets[g] .. prefix_offsets[g + 1], which may cut sequences
 * anywhere; rows of no group have no prefix.  `attn` is as for fa_paged_attn_sm100: its cache's page_table,
 * kv_lens and offsets are those of the sequences' own tokens, and `causal` concerns these alone.  Its
 * workspace takes fa_paged_prefix_workspace_bytes() bytes. */
typedef struct FaPagedPrefixArgs {
  int32_t struct_size; /* sizeof(FaPagedPrefixArgs) */
  FaPagedAttnArgs attn;
  const int32_t* prefix_table;   /* [prefixes, prefix_cols] */
  const int32_t* prefix_offsets; /* [prefixes + 1] */
  const int32_t* prefix_lens;    /* [prefixes] */
  int64_t prefix_stride;         /* elements between the rows of prefix_table */
  int64_t prefix_cols;
  int64_t prefixes;
  int64_t max_prefix_q_len; /* upper bound of a group's rows that the kernel choice goes by (0: total) */
} FaPagedPrefixArgs;

/* Attention of the packed queries over their prefixes and sequences: out, and the logsumexp over both.
 * All else as in fa_paged_attn_sm100. */
FA_API int fa_paged_prefix_sm100(const FaPagedPrefixArgs* args, void* stream);

/* Its workspace, as fa_paged_workspace_bytes. */
FA_API int64_t fa_paged_prefix_workspace_bytes(const FaPagedPrefixArgs* args);

/* The attention weight that cached tokens received.  `weights` [num_pages, heads_kv, page_size] has one
 * float for each (token, kv head) of the cache.  The values of `cache` (v, v_scale) are not read. */
typedef struct FaPagedWeightsArgs {
  int32_t struct_size;     /* sizeof(FaPagedWeightsArgs) */
  const void* q;           /* [total, heads_q, head_dim] */
  const float* lse;        /* [total, heads_q], contiguous: what the attention call over these rows left */
  float* weights;
  void* workspace;         /* fa_paged_weights_workspace_bytes() bytes, 256-byte aligned; needs no clearing */
  int32_t* dev_status;     /* optional device int, 0 on success */
  FaPagedCache cache;
  int64_t q_stride[2];       /* element strides of (row, head); multiples of 16 bytes */
  int64_t weights_stride[2]; /* element strides of (page, head); multiples of 16 bytes */
  int64_t total;
  int64_t heads_q;   /* a multiple of heads_kv */
  int64_t max_q_len; /* upper bound of a sequence's new tokens that the tiling goes by (0: total); a longer
                        sequence is computed all the same */
  int64_t workspace_bytes;
  int32_t dtype;     /* of q: the cache's own, or fp16 / bf16 with a float8 cache */
  int32_t causal;    /* a token gives weight to positions up to its own; 0: to the whole sequence */
  int32_t reset_new; /* the weights of the sequences' new tokens start from 0 */
  float sm_scale;
} FaPagedWeightsArgs;

/* For each sequence, kv head and position: weights += the sum of exp(sm_scale q k - lse) over the rows
 * that attend to it and share the head.  A row with lse = -inf gives nothing, whatever q holds.  Sequences with new tokens
 * only; pages must not belong to two sequences of a call. */
FA_API int fa_paged_weights_sm100(const FaPagedWeightsArgs* args, void* stream);

/* Its workspace, as fa_paged_workspace_bytes. */
FA_API int64_t fa_paged_weights_workspace_bytes(const FaPagedWeightsArgs* args);

/* Eviction by accumulated attention weight, per sequence and kv head.  `weights` [num_pages, heads_kv,
 * page_size] has one float for each (token, kv head) of the cache.  The offsets of `cache` are not read. */
typedef struct FaPagedEvictArgs {
  int32_t struct_size;     /* sizeof(FaPagedEvictArgs) */
  float* weights;          /* moved along with the tokens */
  int32_t* new_lens;       /* [seqs]: min(kv_lens, keep) */
  int32_t* kept;           /* [seqs, heads_kv, keep]: the positions that stay, in order, -1 behind them */
  void* workspace;         /* fa_paged_evict_workspace_bytes() bytes, 256-byte aligned; needs no clearing */
  int32_t* dev_status;     /* optional device int, 0 on success */
  FaPagedCache cache;
  int64_t weights_stride[2]; /* element strides of (page, head); multiples of 16 bytes */
  const int32_t* to_table;   /* [seqs, to_cols]: pages that receive what stays, unless in_place */
  int64_t to_stride;
  int64_t to_cols;
  int64_t keep;     /* tokens that stay of a longer sequence */
  int64_t recent;   /* the last ones, which stay whatever their weight; at most keep */
  int64_t workspace_bytes;
  int32_t in_place; /* what stays goes to the front of the sequence's own pages */
} FaPagedEvictArgs;

/* Of each sequence longer than `keep` every kv head keeps its last `recent` tokens and, of the others, the
 * keep - recent with the largest weights: of equal ones the earlier, and NaN before all.  They keep their
 * order and go to positions 0 .. keep - 1, in K, V, the scales of a float8 cache and the weights.  What
 * lies behind the new length is left as it was.  Shorter sequences stay as they are (not in place: they
 * are copied).  Pages that receive tokens must not belong to another sequence too; those of to_table must
 * not be among those of page_table.  A to_table with fewer places than a sequence has tokens to stay is reported
 * through the device status, and that sequence's results are undefined. */
FA_API int fa_paged_evict_sm100(const FaPagedEvictArgs* args, void* stream);

/* Its workspace, as fa_paged_workspace_bytes. */
FA_API int64_t fa_paged_evict_workspace_bytes(const FaPagedEvictArgs* args);

#ifdef __cplusplus
}
#endif

#endif /* FA_PAGED_SM100_H_ */
