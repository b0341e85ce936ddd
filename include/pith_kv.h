/*
 * pith_kv.h — flat C ABI of libpith_hip.so, third part: the key-value cache of the GQA layer, attention of new tokens to it, and the bookkeeping of a step.
 *
 * What a layer of pithtrain/models/qwen3_30b_a3b.py:384-442 runs when it answers instead of being trained. A token leaves behind a normalised, rotated
 * key and a value for each of its key-value heads, in pages of a cache that all sequences share; new tokens attend to the rows of their sequence, to all of
 * them or to the pages that a cheap score selects for each.
 *
 * The conventions of pith_hip.h hold: status codes, borrowed device pointers, nothing allocated or kept, work enqueued on `stream` only, strides
 * in elements, base-2 LSE. The size of every array that a kernel indexes by data (pages, tables, token counts) is part of the call, and what lies
 * outside is clamped or skipped, so bad values give wrong rows but stay in memory. All counts, lengths, tables and offsets are read by the kernels only: a
 * call that was captured into a graph can be replayed after their contents have changed. They must not change while it runs, and what a call writes must
 * not overlap what it reads, except where that is said.
 */
#ifndef PITH_KV_H
#define PITH_KV_H

#include "pith_hip.h"
#include "pith_latent.h" /* PITH_FP8_E4M3 */

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this part, numbered like PITH_VERSION and independent of it. */
#define PITH_KV_VERSION 100
int pith_kv_version(void);

/* The cache: `pages` pages of page_size rows (a power of two from 16 to 65536; fewer than 2^31 rows in all) of `heads` key-value heads of `dim` features
 * (64 or 128). Row r of head h of page p holds
 *   k + p*k_ps + (h*page_size + r)*dim   bf16, or e4m3 with k_scale + p*k_scale_ps + h*page_size + r (fp32): the feature is value * scale of its row
 *   v                                    likewise
 * so the rows of a head lie one behind the other in a page. Page strides in elements (not used where there is one page); pointers and page strides keep
 * 16-byte alignment (scales: 4 bytes). Slot s is row s % page_size of page s / page_size. */
typedef struct {
  void* k;
  void* v;
  float* k_scale; /* PITH_FP8_E4M3 only */
  float* v_scale;
  int64_t pages, page_size, heads, dim;
  int64_t k_ps, v_ps, k_scale_ps, v_scale_ps;
  int32_t dtype; /* PITH_BF16 | PITH_FP8_E4M3 */
  int32_t reserved0;
} pith_kv_cache;

/* ------------------------------------------------------------------------------------------
 * The bookkeeping of a step, for this cache and the latent one alike: token offsets, positions and slots of the new rows of B requests, and the pages that
 * they need, out of a pool. With c = counts[i] and L = lengths[i] (rows cached before the step):
 *   c < 0    the request has ended: its ceil(L / page_size) pages, in the order of its table, are laid on the pool, its length becomes 0
 *   c >= 0   it gets rows L .. L+c-1. Pages that these need beyond the ceil(L / page_size) it has are taken off the top of the pool (what was laid there in
 *            this call included) and written into its table, or none of them is: where the pool does not suffice for it or for a request in front of it, or
 *            its table is too narrow, granted[i] is 0, its length stays, and its tokens have slots of -1
 * The pool: free_pages [pool_size] int32, of which the first free_count[0] are free, the last of them the top. What ended requests would lay beyond
 * pool_size is dropped.
 * Results: cu_q [B+1] int32, offsets of the tokens (c of each request with c > 0, granted or not; what goes beyond T is cut off, from its request's rows
 * too); position_ids [T] int64 (L + i) and slots [T] int64 of each token, those behind cu_q[B] with position 0 and slot -1; granted [B] int32, rows;
 * lengths_out [B] int32 and free_count_out [1] int32, the values behind the step, which may be lengths and free_count themselves.
 * counts, lengths [B] int32, page_table [B, table_width] int32 (row stride table_rs), updated in place like free_pages. Lengths are taken to be within
 * 0 .. table_width * page_size.
 * workspace: pith_plan_step_workspace_bytes of the same arguments (0 for few tokens and requests), 16-byte aligned, used by the call's kernels only. */
typedef struct {
  const int32_t* counts;
  const int32_t* lengths;
  int32_t* page_table;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* cu_q;
  int64_t* position_ids;
  int64_t* slots;
  int32_t* granted;
  int32_t* lengths_out;
  int32_t* free_count_out;
  void* workspace;
  int64_t workspace_bytes;
  int64_t B, T, table_rs, table_width, pool_size, page_size;
} pith_plan_step_args;

int64_t pith_plan_step_workspace_bytes(const pith_plan_step_args* args);
int pith_plan_step(const pith_plan_step_args* args, pith_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * New tokens (q_norm, k_norm and the rotation, qwen3_30b_a3b.py:417-421, and what a cache keeps of them):
 *     n(x, w) = x * rsqrt(mean(x^2) + eps) * w per head (no weights: x), rot as in pith_norm_rope_args with row position_ids[t] of the tables
 *     q_out[t] = rot(n(q[t], q_weight));   K[slot] = rot(n(k[t], k_weight)),   V[slot] = v[t]
 *     bf16 cache: rounded once;   fp8 cache: s = max|x| / 448 of a row of a head, e4m3(x / s), its scale s (all 0 where x is)
 * q [T, H, dim], k, v [T, heads, dim], q_out [T, H, dim] bf16 with unit stride along the features, token and head strides multiples of 8; q_out may be q
 * itself. Weights [dim] (both or none); cos, sin [P, dim] bf16 tables; position_ids, slots [T] int64. Positions are clamped to the tables, keys and values
 * of tokens whose slot is negative or beyond the cache are skipped (padding). Two tokens of a call must not name the same slot: their rows would mix. T = 0
 * does nothing. */
typedef struct {
  const void* q;
  const void* k;
  const void* v;
  const void* q_weight;
  const void* k_weight;
  const void* cos;
  const void* sin;
  const int64_t* position_ids;
  const int64_t* slots;
  void* q_out;
  int64_t T, P, H;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, q_out_ts, q_out_hs;
  float eps;
  int32_t weight_dtype; /* PITH_BF16 | PITH_F32 */
  pith_kv_cache cache;
} pith_kv_append_args;

int pith_kv_append(const pith_kv_append_args* args, pith_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * Attention of the newest tokens of B sequences to their cached rows, those of the tokens themselves included (append them first). With g = h / (H / heads):
 *     s[t,h,j] = scale * q[t,h] . K[g]_j    over the keys j that token t sees
 *     o[t,h] = softmax(s) V[g],  lse[h,t] = log2 sum_j exp(s)
 * Tokens cu_q[b] .. cu_q[b+1]-1 are sequence b's, its last n = cu_q[b+1]-cu_q[b] rows of lengths[b] (cu_q NULL: one token a sequence, T = B). Token i of
 * them sees rows up to lengths[b]-n+i (causal); with tree_mask all rows in front of the n newest, and of those row j where bit j of tree_mask[token] is set
 * (sequences with n > 64 are then computed with their first 64 new rows visible by bits and none behind: keep n <= 64). A token that sees nothing gets
 * o = 0 and lse = -inf. Tokens from cu_q[B] on are left alone. Lengths are clamped to table_width * page_size, page numbers to the cache, and offsets of
 * cu_q count as their maximum so far, so that a token belongs to one sequence.
 * head_tables = 0: page_table [B, table_width] (row stride table_rs) and lengths [B] are those of all heads. head_tables = 1: page_table
 * [B, heads, table_width] (strides table_rs, table_hs) and lengths [B, heads]: every key-value head has rows of its own, as pith_kv_select leaves them
 * (one token a sequence: no cu_q, no tree_mask).
 * q [T,H,dim], o [T,H,dim] bf16 with token and head strides (multiples of 8); lse [H,T] fp32 (head stride lse_hs). H is a multiple of cache.heads.
 * cu_q [B+1], lengths and tables int32; tree_mask [T] int64 or NULL.
 * workspace: pith_kv_attn_workspace_bytes of the same arguments, 256-byte aligned, used by the call's kernels only. Calls that may overlap in time need one
 * each. */
typedef struct {
  const void* q;
  pith_kv_cache cache;
  const int32_t* page_table;
  const int32_t* lengths;
  const int32_t* cu_q;      /* NULL: one token a sequence */
  const int64_t* tree_mask; /* NULL: causal */
  void* o;
  float* lse;
  void* workspace;
  int64_t workspace_bytes;
  int64_t T, B, H, table_rs, table_hs, table_width;
  int64_t q_ts, q_hs, o_ts, o_hs, lse_hs;
  float scale;
  int32_t head_tables;
} pith_kv_attn_args;

int64_t pith_kv_attn_workspace_bytes(const pith_kv_attn_args* args);
/* Query rows to a row block of the kernel that such a call takes, 16, 32 or 64; 0 for a call that launches nothing or is rejected for its sizes. A row's
 * keys are cut, and its sums ordered, by that and by the lengths of all sequences of the call. In blocks of 16 rows a softmax weight keeps 16 bits in the product with
 * the values (2^-15 of it is lost at most), in those of 32 and 64 the 8 of a bf16 number (2^-8). */
int pith_kv_attn_rows(const pith_kv_attn_args* args);
int pith_kv_attn(const pith_kv_attn_args* args, pith_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * Which pages a token attends to. bounds [pages, heads, 2, dim] bf16 (page stride bounds_ps, a multiple of 8) beside a cache hold the least and the largest
 * value of each key feature over the rows of a page (of e4m3: value * scale; rounded to bf16; NaN where a key has one).
 *   pith_kv_bounds   writes those of every page whose last row is one of the newest tokens of its sequence (T, B, cu_q, lengths, page_table as in
 *                    pith_kv_attn_args, offsets counted likewise; append them first). Others keep what they hold.
 *   pith_kv_select   for token t, which sees n rows (as in the causal pith_kv_attn) in ceil(n / page_size) pages, and each key-value head: all of them if
 *                    they are at most `keep`; else the token's own, the last, and the keep - 1 of the others with the largest scores
 *                        max over the heads h of the group of sum_d max(q[t,h,d] * least_d, q[t,h,d] * largest_d)   (no q . k of the page exceeds
 *                        it, but for the rounding of bounds of e4m3 keys)
 *                    summed in fp64, rounded to fp32 and compared so; equal scores in favour of the page that comes first, NaN above all. Their numbers go, in
 *                    the order of the sequence, to table_out [T, heads, keep] int32 (contiguous; -1 behind the last) and the rows they make to lengths_out
 *                    [T, heads]: a call of pith_kv_attn with head_tables and without cu_q. Tokens that are no sequence's (in front of
 *                    cu_q[0], behind cu_q[B]) and those that see nothing get no page.
 * q [T, H, dim] bf16 as in pith_kv_attn_args. keep >= 1; pith_kv_select takes page tables of up to 16384 pages. Its workspace:
 * pith_kv_select_workspace_bytes (64 MB at most, or what one token needs: more tokens than that serves are taken in parts), 256-byte aligned. */
typedef struct {
  pith_kv_cache cache;
  void* bounds;
  const int32_t* page_table;
  const int32_t* lengths;
  const int32_t* cu_q; /* NULL: one token a sequence */
  int64_t T, B, table_rs, table_width, bounds_ps;
} pith_kv_bounds_args;

int pith_kv_bounds(const pith_kv_bounds_args* args, pith_stream_t stream);

typedef struct {
  const void* q;
  const void* bounds;
  const int32_t* page_table;
  const int32_t* lengths;
  const int32_t* cu_q; /* NULL: one token a sequence */
  int32_t* table_out;
  int32_t* lengths_out;
  void* workspace;
  int64_t workspace_bytes;
  int64_t T, B, H, heads, dim, pages, page_size, keep;
  int64_t q_ts, q_hs, table_rs, table_width, bounds_ps;
} pith_kv_select_args;

int64_t pith_kv_select_workspace_bytes(const pith_kv_select_args* args);
int pith_kv_select(const pith_kv_select_args* args, pith_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* PITH_KV_H */
