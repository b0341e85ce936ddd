/*
 * pith_latent.h — flat C ABI of libpith_hip.so, second part: the MLA layer's latent cache and the absorbed form of its attention.
 *
 * What a layer of pithtrain/models/deepseek_v2_lite.py:420-470 runs when it answers instead of being trained. A token leaves behind one latent
 * vector c (512 features, normalised) and one rotated key part p (64 features), both shared by all heads. The key of head h is
 * [W_uk[h] c | p], its value W_uv[h] c (kv_b_proj, :431-437). Since q . (W_uk c) = (W_uk^T q) . c, queries can be taken into the latent space
 * once and attend to the cached rows themselves, with the sum of the rows as the result: keys and values are never expanded.
 *
 * The conventions of pith_hip.h hold: status codes, borrowed device pointers, nothing allocated or kept, work enqueued on `stream` only, strides
 * in elements, base-2 LSE. The size of every array that a kernel indexes by data (pages, tables, token counts) is part of the call, and what lies
 * outside is clamped or skipped, so bad values give wrong rows but stay in memory.
 */
#ifndef PITH_LATENT_H
#define PITH_LATENT_H

#include "pith_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this part, numbered like PITH_VERSION and independent of it. */
#define PITH_LATENT_VERSION 100
int pith_latent_version(void);

enum { PITH_LATENT_DIM = 512, PITH_LATENT_ROPE_DIM = 64, PITH_LATENT_NOPE_DIM = 128, PITH_LATENT_VALUE_DIM = 128 };
enum { PITH_FP8_E4M3 = 2 }; /* beside PITH_BF16 and PITH_F32 */

/* The cache: `pages` pages of page_size rows (a power of two from 16 to 65536; fewer than 2^31 rows in all). Row r of page p holds
 *   latent + p*latent_ps + r*512   bf16, or e4m3 with scale + p*scale_ps + r (fp32): the feature is value * scale of its row
 *   k_pe   + p*k_pe_ps   + r*64    bf16
 * Page strides in elements (not used where there is one page); pointers and page strides keep 16-byte alignment (scale: 4 bytes). Slot s is row
 * s % page_size of page s / page_size. */
typedef struct {
  void* latent;
  void* k_pe;
  float* scale;  /* PITH_FP8_E4M3 only */
  int64_t pages, page_size;
  int64_t latent_ps, k_pe_ps, scale_ps;
  int32_t dtype; /* of latent: PITH_BF16 | PITH_FP8_E4M3 */
  int32_t reserved0;
} pith_latent_cache;

/* ------------------------------------------------------------------------------------------
 * New tokens into the cache (kv_a_layernorm and the rotation of k_pe, deepseek_v2_lite.py:430-447, and what a cache keeps of them):
 *     n = c * rsqrt(mean(c^2) + eps) * weight        c = kv_a[t, :512]
 *     bf16 cache: latent[slot] = n;   fp8 cache: s = max|n| / 448, latent[slot] = e4m3(n / s), scale[slot] = s (all 0 where n is)
 *     k_pe[slot] = rot(kv_a[t, 512:])                the rotation of pith_mla_assemble_args
 * kv_a [T, 576] bf16 (row stride kv_a_rs, a multiple of 8); weight [512]; cos, sin [P, 64] bf16 tables; position_ids, slots [T] int64. Positions
 * are clamped to the tables, tokens whose slot is negative or beyond the cache are skipped (padding). Two tokens of a call must not name the same
 * slot: their rows would mix. T = 0 does nothing. */
typedef struct {
  const void* kv_a;
  const void* weight;
  const void* cos;
  const void* sin;
  const int64_t* position_ids;
  const int64_t* slots;
  int64_t T, P, kv_a_rs;
  float eps;
  int32_t weight_dtype; /* PITH_BF16 | PITH_F32 */
  pith_latent_cache cache;
} pith_latent_append_args;

int pith_latent_append(const pith_latent_append_args* args, pith_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * Cached rows of B sequences, one behind the other, as bf16 (value * scale, rounded once): what the expanded form of a prompt behind a cached
 * prefix reads (kv_b_proj of them gives keys in two parts and values for pith_attn_fwd without a mask). Sequence b's rows 0 ..
 * cu_rows[b+1]-cu_rows[b]-1 lie in the pages page_table[b, :] (int32, row stride table_rs, table_width entries) and go to output rows cu_rows[b] ..;
 * cu_rows [B+1] int32 ascending from 0. Output rows from cu_rows[B] up to `rows` are left alone. */
typedef struct {
  pith_latent_cache cache;
  const int32_t* page_table;
  const int32_t* cu_rows;
  void* latent_out; /* [rows, 512] bf16, row stride latent_rs */
  void* k_pe_out;   /* [rows, 64] bf16, row stride k_pe_rs */
  int64_t B, rows, table_rs, table_width;
  int64_t latent_rs, k_pe_rs;
} pith_latent_gather_args;

int pith_latent_gather(const pith_latent_gather_args* args, pith_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * The products around the attention. weight [H, 256, 512] bf16 contiguous is kv_b_proj.weight (rows 0..127 of a head W_uk, 128..255 W_uv).
 *   query: q_latent[t,h,:] = sum_d q[t,h,d] weight[h,d,:] (d < 128),  q_pe[t,h,:] = rot(q[t,h,128:])
 *   value: o[t,h,v] = sum_r x[t,h,r] weight[h,128+v,r]
 * x is q [T,H,192] or the latent result [T,H,512], out q_latent [T,H,512] or o [T,H,128], q_pe [T,H,64]; bf16, unit stride along the features,
 * token and head strides (multiples of 8) given. fp32 sums, rounded once. T = 0 does nothing. */
typedef struct {
  const void* x;
  const void* weight;
  void* out;
  void* q_pe;                 /* query only, like what follows */
  const void* cos;
  const void* sin;
  const int64_t* position_ids; /* [T] int64, clamped to the tables */
  int64_t T, H, P;
  int64_t x_ts, x_hs, out_ts, out_hs, q_pe_ts, q_pe_hs;
} pith_latent_absorb_args;

int pith_latent_absorb_query(const pith_latent_absorb_args* args, pith_stream_t stream);
int pith_latent_absorb_value(const pith_latent_absorb_args* args, pith_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * Attention of the newest tokens of B sequences to their cached rows, those of the tokens themselves included (append them first):
 *     s[t,h,j] = scale * (q_latent[t,h] . c_j + q_pe[t,h] . p_j)    over the keys j that token t sees
 *     o[t,h] = softmax(s) c,  lse[h,t] = log2 sum_j exp(s)
 * Tokens cu_q[b] .. cu_q[b+1]-1 are sequence b's, its last n = cu_q[b+1]-cu_q[b] rows of lengths[b]. Token i of them sees rows up to
 * lengths[b]-n+i (causal); with tree_mask all rows in front of the n newest, and of those row j where bit j of tree_mask[token] is set (sequences
 * with n > 64 are then computed with their first 64 new rows visible by bits and none behind: keep n <= 64). A token that sees nothing gets o = 0
 * and lse = -inf. Tokens from cu_q[B] on are left alone. Lengths are clamped to table_width * page_size, page numbers to the cache, and offsets of
 * cu_q count as their maximum so far, so that a token belongs to one sequence.
 * q_latent [T,H,512], q_pe [T,H,64], o [T,H,512] bf16 with token and head strides (multiples of 8); lse [H,T] fp32 (head stride lse_hs).
 * lengths [B], cu_q [B+1], page_table [B, table_width] int32; tree_mask [T] int64 or NULL. All of them are read by the kernels only: a call that
 * was captured into a graph can be replayed after their contents, and those of the cache, have changed. They must not change while it runs, and o
 * and lse must not overlap what it reads.
 * workspace: pith_latent_attn_workspace_bytes of the same arguments, 256-byte aligned, used by the call's kernels only. Calls that may overlap in
 * time need one each. */
typedef struct {
  const void* q_latent;
  const void* q_pe;
  pith_latent_cache cache;
  const int32_t* page_table;
  const int32_t* lengths;
  const int32_t* cu_q;
  const int64_t* tree_mask; /* NULL: causal */
  void* o;
  float* lse;
  void* workspace;
  int64_t workspace_bytes;
  int64_t T, B, H, table_rs, table_width;
  int64_t q_ts, q_hs, q_pe_ts, q_pe_hs, o_ts, o_hs, lse_hs;
  float scale;
  int32_t reserved0;
} pith_latent_attn_args;

int64_t pith_latent_attn_workspace_bytes(const pith_latent_attn_args* args);
/* Query rows to a workgroup of the kernel that such a call takes, 16 or 64; 0 for a call that launches nothing or is rejected for its sizes. A row's
 * keys are cut, and its sums ordered, by that and by the lengths of all sequences of the call. */
int pith_latent_attn_rows(const pith_latent_attn_args* args);
int pith_latent_attn(const pith_latent_attn_args* args, pith_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* PITH_LATENT_H */
