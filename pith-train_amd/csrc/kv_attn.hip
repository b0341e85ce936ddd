// Attention of new tokens to the rows of a key-value cache (include/pith_kv.h).
#include "kv_common.h"

namespace pith {
namespace {

struct KVAttnParams {
  const __bf16* q;
  KVCache cache;
  const int32_t *table, *lengths, *cu_q;
  const int64_t* tree;
  __bf16* o;
  float* lse;
  int64_t table_rs, table_hs, q_ts, q_hs, o_ts, o_hs, lse_hs;
  int T, B, H, group, table_width, head_tables;
  float kappa;  // scale * log2(e)
};

// A wave for every token and query head, a key after the other.
template <int D, bool FP8>
__global__ __launch_bounds__(64) void kv_attn_kernel(KVAttnParams p) {
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, head = h / p.group;
  int seq = t, first = t, n = 1;
  if (p.cu_q) {  // offsets count as their maximum so far
    int most = min(max(p.cu_q[0], 0), p.T);
    for (seq = 0; seq < p.B; ++seq) {
      first = most;
      most = max(most, min(max(p.cu_q[seq + 1], 0), p.T));
      if (t >= first && t < most) break;
    }
    if (seq == p.B) return;
    n = most - first;
  }
  const int length = min(max(p.lengths[p.head_tables ? seq * p.cache.heads + head : seq], 0), p.table_width << p.cache.page_shift);
  const int32_t* const table = p.table + seq * p.table_rs + head * p.table_hs;
  const uint64_t word = p.tree ? (uint64_t)p.tree[t] : 0;
  constexpr int E = D / 64;
  float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) q[e] = (float)p.q[t * p.q_ts + h * p.q_hs + E * lane + e];
  for (int j = 0; j < length; ++j) {
    const int draft = j - (length - n);
    const bool seen = p.tree ? draft < 0 || (draft < 64 && ((word >> (draft & 63)) & 1)) : draft <= t - first;
    if (!seen) continue;
    const int64_t page = safe_page(table[j >> p.cache.page_shift], p.cache.pages);
    const int64_t row = ((int64_t)head << p.cache.page_shift) + (j & ((1 << p.cache.page_shift) - 1));
    float k[E], v[E];
    for (int e = 0; e < E; ++e) {
      if constexpr (FP8) {
        k[e] = (float)fp8x2_to_bf16<false>((uint8_t)p.cache.k[page * p.cache.k_ps + row * D + E * lane + e])[0] * p.cache.k_scale[page * p.cache.k_scale_ps + row];
        v[e] = (float)fp8x2_to_bf16<false>((uint8_t)p.cache.v[page * p.cache.v_ps + row * D + E * lane + e])[0] * p.cache.v_scale[page * p.cache.v_scale_ps + row];
      } else {
        k[e] = (float)reinterpret_cast<const __bf16*>(p.cache.k + page * p.cache.k_ps)[row * D + E * lane + e];
        v[e] = (float)reinterpret_cast<const __bf16*>(p.cache.v + page * p.cache.v_ps)[row * D + E * lane + e];
      }
    }
    float s = 0.f;
    for (int e = 0; e < E; ++e) s += q[e] * k[e];
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    s *= p.kappa;
    const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m - ref), w = __builtin_amdgcn_exp2f(s - ref);
    l = l * alpha + w;
    for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + w * v[e];
    m = top;
  }
  for (int e = 0; e < E; ++e) p.o[t * p.o_ts + h * p.o_hs + E * lane + e] = (__bf16)(l == 0.f ? 0.f : o[e] / l);
  if (lane == 0) p.lse[h * p.lse_hs + t] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
}

int check_attn(const pith_kv_attn_args* a, const char* who) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (const int rc = check_cache(a->cache, who)) return rc;
  if (const int rc = check_table(a->T, a->B, a->cache.heads, a->table_width, a->cache.page_size, !a->cu_q, who)) return rc;
  if (a->H < 1 || a->H > 1024 || a->H % a->cache.heads)
    return fail(PITH_ERR_BAD_SHAPE, "%s: %lld query heads (at most 1024) of %lld key-value heads", who, (long long)a->H, (long long)a->cache.heads);
  if (a->head_tables && a->tree_mask) return fail(PITH_ERR_UNSUPPORTED, "%s: tables of the heads go with causal attention", who);
  return PITH_OK;
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int64_t pith_kv_attn_workspace_bytes(const pith_kv_attn_args* a) {
  if (check_attn(a, "pith_kv_attn_workspace_bytes") != PITH_OK || a->T == 0 || a->B == 0) return 0;
  return 256;
}

extern "C" int pith_kv_attn(const pith_kv_attn_args* a, pith_stream_t stream) {
  const char* who = "pith_kv_attn";
  if (const int rc = check_attn(a, who)) return rc;
  if (a->T == 0 || a->B == 0) return PITH_OK;
  if (!a->q || !a->lengths || !a->o || !a->lse || !a->workspace || (!a->page_table && a->table_width > 0))
    return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if (a->table_width == 0) return fail(PITH_ERR_BAD_SHAPE, "%s: an empty page table holds no rows", who);
  const int64_t dim = a->cache.dim, heads = a->cache.heads;
  if ((a->B > 1 && a->table_rs < a->table_width) || (a->head_tables && heads > 1 && a->table_hs < a->table_width) || (a->T > 1 && (a->q_ts < dim || a->o_ts < dim)) ||
      (a->H > 1 && (a->q_hs < dim || a->o_hs < dim || a->lse_hs < a->T)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a stride is shorter than what it steps over", who);
  if (!aligned16(a->q) || !aligned16(a->o) || (a->q_ts | a->q_hs | a->o_ts | a->o_hs) % 8 || (uintptr_t)a->workspace % 256 || (uintptr_t)a->page_table % 4 ||
      (uintptr_t)a->lengths % 4 || (uintptr_t)a->cu_q % 4 || (uintptr_t)a->lse % 4 || (uintptr_t)a->tree_mask % 8)
    return fail(PITH_ERR_MISALIGNED, "%s: queries and results need 16-byte alignment and strides of multiples of 8, the workspace 256-byte alignment", who);
  const int64_t need = pith_kv_attn_workspace_bytes(a);
  if (a->workspace_bytes < need) return fail(PITH_ERR_BAD_SHAPE, "%s: the workspace has %lld bytes, %lld are needed", who, (long long)a->workspace_bytes, (long long)need);
  KVAttnParams p = {};
  p.q = (const __bf16*)a->q; p.cache = to_device(a->cache); p.table = a->page_table; p.lengths = a->lengths; p.cu_q = a->cu_q; p.tree = a->tree_mask;
  p.o = (__bf16*)a->o; p.lse = a->lse;
  p.table_rs = a->B > 1 ? a->table_rs : 0; p.table_hs = a->head_tables && heads > 1 ? a->table_hs : 0;
  p.q_ts = a->q_ts; p.q_hs = a->q_hs; p.o_ts = a->o_ts; p.o_hs = a->o_hs; p.lse_hs = a->lse_hs;
  p.T = (int)a->T; p.B = (int)a->B; p.H = (int)a->H; p.group = (int)(a->H / heads); p.table_width = (int)a->table_width; p.head_tables = a->head_tables != 0;
  p.kappa = a->scale * 1.4426950408889634f;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)a->T, (unsigned)a->H);
  begin_launch();
  const bool fp8 = a->cache.dtype == PITH_FP8_E4M3;
  if (dim == 128 && fp8) kv_attn_kernel<128, true><<<grid, 64, 0, s>>>(p);
  else if (dim == 128) kv_attn_kernel<128, false><<<grid, 64, 0, s>>>(p);
  else if (fp8) kv_attn_kernel<64, true><<<grid, 64, 0, s>>>(p);
  else kv_attn_kernel<64, false><<<grid, 64, 0, s>>>(p);
  return check_launch(who);
}
