/*
 * C ABI of the serving operators around the sm_100a attention forward (fa2_sm100.h): rotary
 * positions, an 8-bit paged K/V cache that is appended to and read back, and attention of new
 * tokens over it. Extensions: roy6n23/triton-fa2-forward has no counterpart.
 *
 * Built into libfa2_kvcache_sm100.so. Plain pointers, sizes and strides only; every launch is
 * asynchronous on the caller's stream and returns a Fa2Status (fa2_sm100.h). Nothing here
 * allocates device memory.
 *
 * The cache. Codes are e4m3 (sign, 4 exponent bits, 3 mantissa bits, largest value 448), one byte
 * a value, in pages [num_pages, page_size, heads_kv, head_dim]; k_scale and v_scale hold one fp32
 * for each row of head_dim values, [num_pages, page_size, heads_kv]. A row x is stored as
 *     scale = max|x| / 448,  code = e4m3(x / scale) (round to nearest even; a zero row: 0 and 0)
 * and stands for code * scale. A row that holds a NaN or an infinity is stored as codes 0 and a
 * NaN scale, so it reads back as NaN; no code written here is a NaN. Strides are free (page, row,
 * head) as long as every row of codes starts on a 16-byte boundary (and, to be written, the rows lie
 * apart: the dimensions nest, no row is another's memory); pages whose rows of one head
 * are adjacent (head stride = page_size * head_dim) are read fastest.
 *
 * Sequence b's key j is in page block_table[b * block_table_stride + j / page_size], row
 * j % page_size. Table entries past a sequence's last page are not read. Device-side reports go
 * to err_flag as in fa2_sm100.h: FA2_ERR_SHAPE (a length that is negative, longer than the table
 * or the declared maximum, or not covered by its tensor) and FA2_ERR_PAGE (a table entry outside
 * the cache); the row or sequence in question is left out, nothing is accessed out of range. A word
 * that already holds a report changes nothing here; fa2_fwd_sm100's kernels stop for one in theirs,
 * so give these calls another word than those.
 */
#ifndef FA2_KVCACHE_SM100_H_
#define FA2_KVCACHE_SM100_H_

#include <stdint.h>

#include "fa2_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FA2_KVCACHE_ABI_VERSION 1

typedef struct Fa2Kv8Cache {
  void* k; /* e4m3 codes */
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t k_stride[3]; /* elements, order (page, row, head); the d stride is 1 */
  int64_t v_stride[3];
  int64_t ks_stride[3];
  int64_t vs_stride[3];
  int32_t num_pages;
  int32_t page_size; /* 16, 32, 64 or a multiple of 128 */
  int32_t heads_kv;
  int32_t head_dim; /* 16, 32, 64 or 128 */
} Fa2Kv8Cache;

/* Rotary positions of q and (unless k is NULL) k in one launch. For a pair (a, c) of a head's
 * values and the angle t = position * inv_freq[i]:
 *     a' = magnitude * (a cos t - c sin t),  c' = magnitude * (a sin t + c cos t)
 * with -t in place of t when `inverse` (the transposed map: the gradient of the forward one).
 * Pairs are (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when `interleaved`; values from rotary_dim
 * on are copied. out may be in (each value is read before it is written, by the same thread), as long as
 * every value of q and k has memory of its own. */
typedef struct Fa2RotaryParams {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_stride[4]; /* elements, order (b, h, n, d) */
  int64_t k_stride[4];
  int64_t q_out_stride[4];
  int64_t k_out_stride[4];
  const void* positions;  /* int32 or int64, element strides below */
  int64_t pos_stride[2];  /* (b, n) */
  const double* inv_freq; /* radians a position, [rotary_dim / 2] */
  int32_t pos_is_64;
  int32_t batch;
  int32_t seqlen;
  int32_t heads_q;
  int32_t heads_kv; /* 0 when k is NULL */
  int32_t head_dim; /* any size >= 2 */
  int32_t rotary_dim; /* even, <= head_dim */
  int32_t dtype;      /* Fa2DType */
  int32_t interleaved;
  int32_t inverse;
  float magnitude;
  int32_t reserved;
} Fa2RotaryParams;

/* Writes new K/V rows into the cache. Sequence b's n_b new tokens are its last n_b positions:
 * cache_seqlens[b] counts them already. Fixed-length: k, v [B, H, N, D], n_b = seqlen; a sequence
 * with cache_seqlens[b] == 0 is skipped. Packed (cu_seqlens != NULL): k, v [total, H, D] with the
 * token axis as n, n_b = cu_seqlens[b + 1] - cu_seqlens[b]. Two positions written by one call must
 * not share a cache row (a page that two sequences share may be read, not appended to). Sums that
 * fall or go past seqlen are reported; a sequence that goes past it is left out. */
typedef struct Fa2Kv8AppendParams {
  Fa2Kv8Cache cache;
  const void* k;
  const void* v;
  int64_t k_in_stride[4]; /* elements, order (b, h, n, d) */
  int64_t v_in_stride[4];
  const int32_t* block_table;
  const int32_t* cache_seqlens; /* [batch] keys after the append */
  const int32_t* cu_seqlens;    /* packed: [batch + 1]; else NULL */
  int32_t* err_flag;
  int64_t block_table_stride;
  int32_t pages_per_seq;
  int32_t batch;
  int32_t seqlen; /* fixed-length: N; packed: total rows of k and v */
  int32_t dtype;
} Fa2Kv8AppendParams;

/* Reads the first n_b keys of every sequence back into k_out, v_out [total, H, D] (contiguous),
 * n_b = cu_seqlens[b + 1] - cu_seqlens[b]. Rows past cu_seqlens[batch] are left as they were; rows
 * whose page is refused, and those of a sequence that goes past `total`, are zeros. Sums that fall or
 * go past `total` are reported. */
typedef struct Fa2Kv8ReadParams {
  Fa2Kv8Cache cache;
  void* k_out;
  void* v_out;
  const int32_t* block_table;
  const int32_t* cu_seqlens;
  int32_t* err_flag;
  int64_t block_table_stride;
  int32_t pages_per_seq;
  int32_t batch;
  int32_t total;
  int32_t dtype;
} Fa2Kv8ReadParams;

/* out = softmax(q k^T * sm_scale + mask) v over the cache. q, o: [B, H_q, N, D], or packed
 * [total, H_q, D] with cu_seqlens_q (the token axis as n). causal_align as in fa2_sm100.h, per
 * sequence. A query that sees no key gets zeros, and so do those of a sequence whose cache_seqlens entry is
 * refused. Not written: rows of no sequence; rows of one whose number of queries is refused (negative, above
 * seqlen_q, or past total_q); every row that sees a key, where sums that go back and forth make 2^30 units
 * of work or more (FA2_ERR_SHAPE). The sequences of a call share the GPU as one line of work that is cut into
 * equal shares, and partial sums are joined in its order: the same call gives the same bits, but another batch
 * around a sequence may cut it elsewhere and change its last bits. */
typedef struct Fa2Kv8AttnParams {
  Fa2Kv8Cache cache;
  const void* q;
  void* o;
  int64_t q_stride[4]; /* elements, order (b, h, n, d); d stride 1 */
  int64_t o_stride[4];
  const int32_t* block_table;
  const int32_t* cache_seqlens;
  const int32_t* cu_seqlens_q;
  int32_t* err_flag;
  void* workspace; /* fa2_kv8_attn_sm100_workspace_bytes() bytes, 16-byte aligned; not to be shared
                    * by calls that may run at the same time */
  int64_t workspace_bytes;
  int64_t block_table_stride;
  int64_t timeout_cycles; /* per-wait limit in SM clocks; <= 0 selects the default (~1 s) */
  int32_t pages_per_seq;
  int32_t batch;
  int32_t heads_q;
  int32_t seqlen_q;     /* N, or the largest of a packed batch */
  int32_t total_q;      /* packed: rows of q and o */
  int32_t max_seqlen_k; /* upper bound of cache_seqlens (which is 2^31 - 1024 at most) */
  int32_t dtype;
  int32_t causal;
  int32_t causal_align;
  int32_t num_splits; /* 0: chosen from the sizes; else the CTAs that share the work, for each
                       * (sequence, kv head, row block): key ranges where those are alike */
  float qk_scale;     /* sm_scale * log2(e), > 0 */
  int32_t reserved;
} Fa2Kv8AttnParams;

FA2_API int fa2_rotary_sm100_check(const Fa2RotaryParams* p); /* host only, no CUDA calls */
FA2_API int fa2_rotary_sm100(const Fa2RotaryParams* p, void* stream);

FA2_API int fa2_kv8_append_sm100_check(const Fa2Kv8AppendParams* p);
FA2_API int fa2_kv8_append_sm100(const Fa2Kv8AppendParams* p, void* stream);

FA2_API int fa2_kv8_read_sm100_check(const Fa2Kv8ReadParams* p);
FA2_API int fa2_kv8_read_sm100(const Fa2Kv8ReadParams* p, void* stream);

FA2_API int fa2_kv8_attn_sm100_check(const Fa2Kv8AttnParams* p);
/* Workspace of the call `p` describes, which follows from batch, heads, head_dim, seqlen_q, max_seqlen_k
 * and num_splits. Host only; -1 where the check refuses p (the workspace's own fields aside). */
FA2_API int64_t fa2_kv8_attn_sm100_workspace_bytes(const Fa2Kv8AttnParams* p);
FA2_API int fa2_kv8_attn_sm100(const Fa2Kv8AttnParams* p, void* stream);

FA2_API int fa2_kvcache_sm100_abi_version(void);
/* sizeof of the parameter structs, in the order rotary, append, read, attention. */
FA2_API int64_t fa2_kvcache_sm100_params_size(int32_t which);

#ifdef __cplusplus
}
#endif

#endif /* FA2_KVCACHE_SM100_H_ */
