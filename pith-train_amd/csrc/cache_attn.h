// What the kernels of the two caches share: scans and sums over the lanes of a wavefront, softmax references, e4m3.
#pragma once

#include "latent_common.h"

namespace pith {

// Inclusive sums over the lanes of a wavefront.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_dpp(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = add_dpp<0x111, 0xf>(x);  // from 1, 2, 4, 8 lanes below in the row of 16
  x = add_dpp<0x112, 0xf>(x);
  x = add_dpp<0x114, 0xf>(x);
  x = add_dpp<0x118, 0xf>(x);
  x = add_dpp<0x142, 0xa>(x);  // lane 15 of a row to the next row, then lane 31 to the upper half
  return add_dpp<0x143, 0xc>(x);
}

// Inclusive maxima of values from 0 on.
template <int CTRL, int ROWS>
__device__ __forceinline__ int max_dpp(int x) {
  return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_scan_max(int x) {
  x = max_dpp<0x111, 0xf>(x);
  x = max_dpp<0x112, 0xf>(x);
  x = max_dpp<0x114, 0xf>(x);
  x = max_dpp<0x118, 0xf>(x);
  x = max_dpp<0x142, 0xa>(x);
  return max_dpp<0x143, 0xc>(x);
}

// max / sum over the four lanes c, c + 16, c + 32, c + 48 that share a query row
__device__ __forceinline__ float quad_max(float x) {
  const int i = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  return pair_max(fmaxf(__int_as_float(r[0]), __int_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
  const int i = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  return pair_sum(__int_as_float(r[0]) + __int_as_float(r[1]));
}

// Eight e4m3 values (two words) -> bf16, exact.
__device__ __forceinline__ bf16x8 widen(uint32_t w0, uint32_t w1) {
  const bf16x2 a = fp8x2_to_bf16<false>(w0), b = fp8x2_to_bf16<true>(w0), c = fp8x2_to_bf16<false>(w1), d = fp8x2_to_bf16<true>(w1);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Tables that nobody writes while the kernel runs, read as constant memory: by scalar loads, which the counted waits for tiles do not see.
typedef const __attribute__((address_space(4))) int32_t* ScalarTable;

// x *= f in place: as a plain product under a branch the accumulators are copied on the other way, which doubles their registers. The compiler does not
// look into the statement for hazards: f may come from v_exp_f32 right before it (one wait state), and x from products of the tile before, which have ended: they stand
// two barriers away, or in front of the products whose scores f comes from.
__device__ __forceinline__ void scale_in_place(f32x4& x, float f) {
  float a = x[0], b = x[1], c = x[2], d = x[3];
  asm("s_nop 1\n\tv_mul_f32 %0, %4, %0\n\tv_mul_f32 %1, %4, %1\n\tv_mul_f32 %2, %4, %2\n\tv_mul_f32 %3, %4, %3" : "+v"(a), "+v"(b), "+v"(c), "+v"(d) : "v"(f));
  x = f32x4{a, b, c, d};
}

// Where a score may exceed the reference of its row's weights, in bits, before the reference is moved: weights stay below 2^8, far from the end of
// their range, and neither they nor the sums lose precision by it.
constexpr float kSlack = 8.f;
// A row's reference behind scores of up to `top`; it stands unless they are beyond the slack, whatever other rows do (no row's result depends on another's).
__device__ __forceinline__ float moved(float reference, float top) { return top > reference + kSlack ? top : reference; }

}  // namespace pith
