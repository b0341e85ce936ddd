// What the kernels of the key-value cache (include/pith_kv.h) share.
#pragma once

#include "cache_attn.h"
#include "latent_common.h"
#include "pith_kv.h"

namespace pith {

struct KVCache {
  char* k;
  char* v;
  float* k_scale;
  float* v_scale;
  int64_t k_ps, v_ps;              // bytes
  int64_t k_scale_ps, v_scale_ps;  // elements
  int pages, page_shift, heads;
};

inline KVCache to_device(const pith_kv_cache& c) {
  KVCache d = {};
  const int64_t element = c.dtype == PITH_FP8_E4M3 ? 1 : 2;
  d.k = (char*)c.k; d.v = (char*)c.v; d.k_scale = c.k_scale; d.v_scale = c.v_scale;
  d.k_ps = c.k_ps * element; d.v_ps = c.v_ps * element; d.k_scale_ps = c.k_scale_ps; d.v_scale_ps = c.v_scale_ps;
  d.pages = (int)c.pages; d.heads = (int)c.heads;
  d.page_shift = __builtin_ctzll((unsigned long long)c.page_size);
  return d;
}

// A value of another lane of the row of 16.
template <int CTRL>
__device__ __forceinline__ float lane_dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140, kDppRotate8 = 0x128, kDppQuadMirror = 0x1B;
// Over groups of 8 or 16 lanes; all of a group have the result. (Behind the first two steps lanes of a quad agree, so a mirrored half or row is as good as an
// exchanged one.)
template <int LANES, typename F>
__device__ __forceinline__ float group_reduce(float x, const F& f) {
  static_assert(LANES == 8 || LANES == 16, "rows of 64 or 128 features");
  x = f(x, lane_dpp<kDppXor1>(x));
  x = f(x, lane_dpp<kDppXor2>(x));
  x = f(x, lane_dpp<kDppHalfMirror>(x));
  if constexpr (LANES == 16) x = f(x, lane_dpp<kDppMirror>(x));
  return x;
}
// Of the lane half a group away.
template <int LANES>
__device__ __forceinline__ float other_half(float x) {
  if constexpr (LANES == 16) return lane_dpp<kDppRotate8>(x);
  else return lane_dpp<kDppQuadMirror>(lane_dpp<kDppHalfMirror>(x));
}

// Sizes of pages, heads and features, of a cache or of the bounds beside one.
inline int check_pages(int64_t pages, int64_t page_size, int64_t heads, int64_t dim, const char* who) {
  if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: page size %lld is not a power of two from 16 to 65536", who, (long long)page_size);
  if (pages < 1 || pages > ((int64_t)1 << 31) / page_size - 1)
    return fail(PITH_ERR_BAD_SHAPE, "%s: %lld pages of %lld rows: at least one, and fewer than 2^31 rows", who, (long long)pages, (long long)page_size);
  if (heads < 1 || heads > 1024) return fail(PITH_ERR_BAD_SHAPE, "%s: %lld key-value heads (1 to 1024)", who, (long long)heads);
  if (dim != 64 && dim != 128) return fail(PITH_ERR_UNSUPPORTED, "%s: heads of %lld features (64 or 128)", who, (long long)dim);
  return PITH_OK;
}

inline int check_cache(const pith_kv_cache& c, const char* who) {
  if (c.dtype != PITH_BF16 && c.dtype != PITH_FP8_E4M3) return fail(PITH_ERR_BAD_DTYPE, "%s: cache dtype %d is neither bf16 nor e4m3", who, c.dtype);
  const bool fp8 = c.dtype == PITH_FP8_E4M3;
  if (!c.k || !c.v || (fp8 && (!c.k_scale || !c.v_scale))) return fail(PITH_ERR_NULL_POINTER, "%s: a cache pointer is NULL", who);
  if (const int rc = check_pages(c.pages, c.page_size, c.heads, c.dim, who)) return rc;
  const bool strides = c.pages > 1;  // those of a single page are never used
  const int64_t rows = c.heads * c.page_size;
  if (strides && (c.k_ps < rows * c.dim || c.v_ps < rows * c.dim || (fp8 && (c.k_scale_ps < rows || c.v_scale_ps < rows))))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a page stride is shorter than a page", who);
  const int64_t unit = fp8 ? 16 : 8;
  if (!aligned16(c.k) || !aligned16(c.v) || (strides && (c.k_ps % unit || c.v_ps % unit)) || (fp8 && ((uintptr_t)c.k_scale % 4 || (uintptr_t)c.v_scale % 4)))
    return fail(PITH_ERR_MISALIGNED, "%s: the cache breaks the 16-byte alignment", who);
  return PITH_OK;
}

// Counts of a call that reads page tables.
inline int check_table(int64_t T, int64_t B, int64_t heads, int64_t table_width, int64_t page_size, bool one_each, const char* who) {
  if (T < 0 || B < 0 || T > 1 << 20 || B > 1 << 20 || table_width < 0)
    return fail(PITH_ERR_BAD_SHAPE, "%s: T = %lld, B = %lld (at most 2^20), table_width = %lld", who, (long long)T, (long long)B, (long long)table_width);
  if (one_each && T != B) return fail(PITH_ERR_BAD_SHAPE, "%s: %lld tokens of %lld sequences without cu_q: one token a sequence", who, (long long)T, (long long)B);
  if (table_width > (0x7fffffff - 4096) / page_size) return fail(PITH_ERR_UNSUPPORTED, "%s: page tables of 2^31 rows or more", who);
  return PITH_OK;
}

}  // namespace pith
