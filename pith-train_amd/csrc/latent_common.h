// What the kernels of the latent cache (include/pith_latent.h) share.
#pragma once

#include "attn_tiles.h"
#include "pith_latent.h"

namespace pith {

constexpr int kLatent = PITH_LATENT_DIM, kRope = PITH_LATENT_ROPE_DIM, kNope = PITH_LATENT_NOPE_DIM, kValue = PITH_LATENT_VALUE_DIM;
constexpr float kFp8Max = 448.f;

struct LatentCache {
  char* latent;
  __bf16* k_pe;
  float* scale;
  int64_t latent_ps, k_pe_ps, scale_ps;  // latent_ps in bytes, the others in elements
  int pages, page_shift;
};

inline LatentCache to_device(const pith_latent_cache& c) {
  LatentCache d = {};
  d.latent = (char*)c.latent;
  d.k_pe = (__bf16*)c.k_pe;
  d.scale = c.scale;
  d.latent_ps = c.latent_ps * (c.dtype == PITH_FP8_E4M3 ? 1 : 2);
  d.k_pe_ps = c.k_pe_ps;
  d.scale_ps = c.scale_ps;
  d.pages = (int)c.pages;
  d.page_shift = __builtin_ctzll((unsigned long long)c.page_size);
  return d;
}

inline int check_cache(const pith_latent_cache& c, const char* who) {
  if (c.dtype != PITH_BF16 && c.dtype != PITH_FP8_E4M3) return fail(PITH_ERR_BAD_DTYPE, "%s: cache dtype %d is neither bf16 nor e4m3", who, c.dtype);
  const bool fp8 = c.dtype == PITH_FP8_E4M3;
  if (!c.latent || !c.k_pe || (fp8 && !c.scale)) return fail(PITH_ERR_NULL_POINTER, "%s: a cache pointer is NULL", who);
  if (c.page_size < 16 || c.page_size > 65536 || (c.page_size & (c.page_size - 1)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: page size %lld is not a power of two from 16 to 65536", who, (long long)c.page_size);
  if (c.pages < 1 || c.pages > ((int64_t)1 << 31) / c.page_size - 1)
    return fail(PITH_ERR_BAD_SHAPE, "%s: %lld pages of %lld rows: at least one, and fewer than 2^31 rows", who, (long long)c.pages, (long long)c.page_size);
  const bool strides = c.pages > 1;  // those of a single page are never used
  if (strides && (c.latent_ps < c.page_size * kLatent || c.k_pe_ps < c.page_size * kRope || (fp8 && c.scale_ps < c.page_size)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a page stride is shorter than a page", who);
  if (!aligned16(c.latent) || !aligned16(c.k_pe) || (strides && (c.latent_ps % (fp8 ? 16 : 8) || c.k_pe_ps % 8)) || (fp8 && (uintptr_t)c.scale % 4))
    return fail(PITH_ERR_MISALIGNED, "%s: the cache breaks the 16-byte alignment", who);
  return PITH_OK;
}

// Page number of a table entry, kept inside the cache.
__device__ __forceinline__ int safe_page(int page, int pages) { return min(max(page, 0), pages - 1); }

// Two e4m3 values (the low or the high half of `word`) -> two bf16, exact.
template <bool HIGH>
__device__ __forceinline__ bf16x2 fp8x2_to_bf16(uint32_t word) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.0f, HIGH);
}

// Rotated pair j (0..31) of a rotary vector whose interleaved elements 2j, 2j+1 are `pair` (bf16 x 2): features j and 32 + j of the result.
__device__ __forceinline__ void rotate_pair(uint32_t pair, const __bf16* cos_row, const __bf16* sin_row, int j, float& first, float& second) {
  const float even = bf16lo_to_f32(pair), odd = bf16hi_to_f32(pair);
  first = even * (float)cos_row[j] - odd * (float)sin_row[j];
  second = odd * (float)cos_row[kRope / 2 + j] + even * (float)sin_row[kRope / 2 + j];
}
__device__ __forceinline__ int64_t clamped_position(int64_t pos, int64_t P) { return pos < 0 ? 0 : (pos >= P ? P - 1 : pos); }

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Swizzle of rows that are whole multiples of 256 bytes: piece (16 bytes) q of row r lies at q ^ row_swizzle(r). LDS serves 256 bytes a cycle, and a
// wavefront's 16-byte reads as lanes 0-3 12-15 20-27, then 4-11 16-19 28-31, and the upper half alike (measured with the counter of bank conflicts, two
// lanes at a time on one bank); 8-byte reads as its halves. So the fragment reads of 16x16x32 products (lane c + 16 g: row c, piece q + g) want rows
// {0-3, 12-15} and {4-11} each in pairs that differ in the last bit, and the transposed ones (lane: row 8 g + c / 4 or four more, half a piece of a
// pair) want the pairs of rows {0-3, 8-11} to differ, and of {4-7, 12-15}: this has no conflict in either. (tile_swizzle serves 32-row products.)
__device__ __forceinline__ int row_swizzle(int row) { return ((((row >> 3) ^ (row >> 2)) & 1) << 3) | ((row & 3) << 1) | ((row >> 3) & 1); }

// load_lds16 from an address of each lane's own.
__device__ __forceinline__ void load_lds16_at(const void* src, char* dst_wave) {
  const uint32_t lds_addr = (uint32_t)(uintptr_t)(lds_char*)dst_wave;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(src) : "memory");
}

// The next of a row of load_lds16's: `OFFSET` behind the last one's global base and LDS place alike (M0 stays as that statement left it: nothing else in
// these kernels writes it).
template <int OFFSET>
__device__ __forceinline__ void load_lds16_next(const char* base, int offset) {
  asm volatile("global_load_lds_dwordx4 %0, %1 offset:%2" : : "v"(offset), "s"(base), "n"(OFFSET) : "memory");
}

// Until all but the wave's last LATER requests are there.
template <int LATER>
__device__ __forceinline__ void wait_loads() {
  static_assert(LATER < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (LATER & 15) | ((LATER >> 4) << 14));
  asm volatile("" ::: "memory");
}

// LDS addresses as numbers, for places that are the XOR of a lane's first one and a constant.
__device__ __forceinline__ uint32_t lds_address(const char* x) { return (uint32_t)(uintptr_t)(const lds_char*)x; }
template <typename V>
__device__ __forceinline__ const __attribute__((address_space(3))) V* lds_at(uint32_t address) {
  return (const __attribute__((address_space(3))) V*)(uintptr_t)address;
}

}  // namespace pith
