// The latent cache's rows: written as new tokens come (RMS norm of the latent part, rotation of the rotary part, quantisation), and read back.
//
// Both move memory and little else. A token is one wavefront's work: its 512 latent features are 16 bytes a lane, so a row goes in and out by
// whole 1-KB instructions and its sums stay in registers. 8192 tokens into a bf16 cache 6.5 us (21 MB, 3.3 TB/s: four rounds of loads that wait for one another,
// the slot, the row and the weights behind the branch on it, then, behind the latent row's store, the position and its row of the tables), 32 tokens
// 3.6 us (an empty kernel 2.5); 75000 rows of 16 sequences out of an e4m3 cache 31.6 us (156 MB, 4.9 TB/s, the rate of a large copy), 1021 rows 4.6 us.
#include "latent_common.h"

namespace pith {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m));
  return x;
}

struct AppendParams {
  const __bf16* kv_a;
  const void* weight;
  const __bf16* cos;
  const __bf16* sin;
  const int64_t* pos;
  const int64_t* slots;
  int64_t T, P, kv_a_rs, rows;
  float eps;
  LatentCache cache;
};

// n = c * rsqrt(mean(c^2) + eps) * weight in fp32; bf16 rows are rounded once, e4m3 rows once behind the division by their scale (to nearest even;
// the largest feature becomes +-448 exactly). The scale is the fp32 quotient, not a power of two: it costs nothing where it is applied (a factor of
// the whole row, to the score and to the softmax weight) and keeps up to a bit of precision. (The order of the sum of squares and rsqrtf leave the last bit
// of a feature open in fp32, so one that lies next to the middle of two e4m3 values may go to either.)
template <bool FP8, bool W_F32>
__global__ __launch_bounds__(kThreads) void latent_append_kernel(AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (t >= p.T) return;
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.rows) return;
  const __bf16* row = p.kv_a + t * p.kv_a_rs;
  const u32x4 x = *reinterpret_cast<const u32x4*>(row + 8 * lane);
  const uint32_t pair = lane < kRope / 2 ? *reinterpret_cast<const uint32_t*>(row + kLatent + 2 * lane) : 0;
  float v[8], w[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[2 * e] = bf16lo_to_f32(x[e]), v[2 * e + 1] = bf16hi_to_f32(x[e]);
  if constexpr (W_F32) {
    const f32x4* src = reinterpret_cast<const f32x4*>(p.weight) + 2 * lane;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = src[e >> 2][e & 3];
  } else {
    const u32x4 wb = reinterpret_cast<const u32x4*>(p.weight)[lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[2 * e] = bf16lo_to_f32(wb[e]), w[2 * e + 1] = bf16hi_to_f32(wb[e]);
  }
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum += v[e] * v[e];
  const float inv = rsqrtf(wave_sum(sum) * (1.f / kLatent) + p.eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * w[e];

  const int64_t page = slot >> p.cache.page_shift, in_page = slot & ((1 << p.cache.page_shift) - 1);
  char* const dst = p.cache.latent + page * p.cache.latent_ps;
  if constexpr (FP8) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
    const float scale = wave_max(top) / kFp8Max;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = scale > 0.f ? v[e] / scale : v[e];  // (a row of zeros stays one; NaN stays NaN)
      y[e] = q > kFp8Max ? kFp8Max : (q < -kFp8Max ? -kFp8Max : q);
    }
    u32x2 out;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      int word = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * e], y[4 * e + 1], 0, false);
      word = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * e + 2], y[4 * e + 3], word, true);
      out[e] = (uint32_t)word;
    }
    *reinterpret_cast<u32x2*>(dst + in_page * kLatent + 8 * lane) = out;
    if (lane == 0) p.cache.scale[page * p.cache.scale_ps + in_page] = scale;
  } else {
    u32x4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<u32x4*>(dst + in_page * (2 * kLatent) + 16 * lane) = out;
  }
  if (lane < kRope / 2) {
    const int64_t at = clamped_position(p.pos[t], p.P) * kRope;
    float first, second;
    rotate_pair(pair, p.cos + at, p.sin + at, lane, first, second);
    __bf16* pe = p.cache.k_pe + page * p.cache.k_pe_ps + in_page * kRope;
    pe[lane] = (__bf16)first;
    pe[kRope / 2 + lane] = (__bf16)second;
  }
}

struct GatherParams {
  LatentCache cache;
  const int32_t* table;
  const int32_t* cu_rows;
  __bf16* latent_out;
  __bf16* k_pe_out;
  int64_t table_rs, latent_rs, k_pe_rs;
  int B, rows, table_width;
};

constexpr int kGatherRows = 16;  // of a wave

// A wave looks its rows' sequences up together (lane i: the sequence end i; a row's sequence is the number of ends at or below it), then moves row
// after row.
template <bool FP8>
__global__ __launch_bounds__(kThreads) void latent_gather_kernel(GatherParams p) {
  const int lane = threadIdx.x & 63;
  const int row0 = (blockIdx.x * kWaves + (threadIdx.x >> 6)) * kGatherRows;
  const int total = min(p.cu_rows[p.B], p.rows);
  if (row0 >= total) return;
  const int n = min(kGatherRows, total - row0);
  int seq = 0;  // lane i < 16: of row row0 + i
  const int mine = row0 + min(lane & 15, n - 1);
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int end = b0 + lane < p.B ? p.cu_rows[b0 + lane + 1] : 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kGatherRows; ++i) {
      const int below = __popcll(__ballot(end <= row0 + min(i, n - 1)));
      seq += (lane & 15) == i ? below : 0;
    }
  }
  seq = min(seq, p.B - 1);
  const int at = max(mine - p.cu_rows[seq], 0);
  const int page = safe_page(p.table[seq * p.table_rs + min(at >> p.cache.page_shift, p.table_width - 1)], p.cache.pages);
  const int in_page = at & ((1 << p.cache.page_shift) - 1);

  // eight rows in flight (rows behind the wave's last one are read as that one)
#pragma unroll
  for (int i0 = 0; i0 < kGatherRows; i0 += 8) {
    u32x4 v[8];
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = min(i0 + i, n - 1);
      const int64_t pg = __builtin_amdgcn_readlane(page, k);
      const int r = __builtin_amdgcn_readlane(in_page, k);
      const char* const src = p.cache.latent + pg * p.cache.latent_ps;
      if constexpr (FP8) {
        const u32x2 q = *reinterpret_cast<const u32x2*>(src + (int64_t)r * kLatent + 8 * lane);
        v[i][0] = q[0], v[i][1] = q[1];
        s[i] = p.cache.scale[pg * p.cache.scale_ps + r];
      } else {
        v[i] = *reinterpret_cast<const u32x4*>(src + (int64_t)r * (2 * kLatent) + 16 * lane);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i >= n) break;
      if constexpr (FP8) {
        const u32x2 q = {v[i][0], v[i][1]};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bf16x2 two = (e & 1) ? fp8x2_to_bf16<true>(q[e >> 1]) : fp8x2_to_bf16<false>(q[e >> 1]);
          v[i][e] = pack_bf16x2((float)two[0] * s[i], (float)two[1] * s[i]);
        }
      }
      *reinterpret_cast<u32x4*>(p.latent_out + (int64_t)(row0 + i0 + i) * p.latent_rs + 8 * lane) = v[i];
    }
  }
  // rotary parts: 8 lanes a row, 8 rows an instruction
#pragma unroll
  for (int i0 = 0; i0 < kGatherRows; i0 += 8) {
    const int i = i0 + (lane >> 3);
    const int64_t pg = __shfl(page, i);
    const int r = __shfl(in_page, i);
    if (i < n)
      *reinterpret_cast<u32x4*>(p.k_pe_out + (int64_t)(row0 + i) * p.k_pe_rs + 8 * (lane & 7)) =
          *reinterpret_cast<const u32x4*>(p.cache.k_pe + pg * p.cache.k_pe_ps + (int64_t)r * kRope + 8 * (lane & 7));
  }
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int pith_latent_version(void) { return PITH_LATENT_VERSION; }

extern "C" int pith_latent_append(const pith_latent_append_args* a, pith_stream_t stream) {
  const char* who = "pith_latent_append";
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (a->T < 0 || a->T > 0x7fffffff || a->P < 1) return fail(PITH_ERR_BAD_SHAPE, "%s: T = %lld tokens, tables of %lld positions", who, (long long)a->T, (long long)a->P);
  if (const int rc = check_cache(a->cache, who)) return rc;
  if (a->T == 0) return PITH_OK;
  if (!a->kv_a || !a->weight || !a->cos || !a->sin || !a->position_ids || !a->slots) return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if (a->weight_dtype != PITH_BF16 && a->weight_dtype != PITH_F32) return fail(PITH_ERR_BAD_DTYPE, "%s: weight_dtype %d", who, a->weight_dtype);
  if (a->T > 1 && a->kv_a_rs < kLatent + kRope) return fail(PITH_ERR_BAD_SHAPE, "%s: rows of kv_a overlap", who);
  if (!aligned16(a->kv_a) || a->kv_a_rs % 8 || !aligned16(a->weight) || (uintptr_t)a->cos % 2 || (uintptr_t)a->sin % 2 || (uintptr_t)a->position_ids % 8 || (uintptr_t)a->slots % 8)
    return fail(PITH_ERR_MISALIGNED, "%s: kv_a and weight need 16-byte alignment, position_ids and slots 8-byte", who);
  AppendParams p = {};
  p.kv_a = (const __bf16*)a->kv_a; p.weight = a->weight; p.cos = (const __bf16*)a->cos; p.sin = (const __bf16*)a->sin;
  p.pos = a->position_ids; p.slots = a->slots; p.T = a->T; p.P = a->P; p.kv_a_rs = a->kv_a_rs; p.eps = a->eps;
  p.rows = a->cache.pages * a->cache.page_size;
  p.cache = to_device(a->cache);
  const dim3 grid((unsigned)((a->T + kWaves - 1) / kWaves));
  begin_launch();
  const bool fp8 = a->cache.dtype == PITH_FP8_E4M3, f32 = a->weight_dtype == PITH_F32;
  if (fp8 && f32) latent_append_kernel<true, true><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
  else if (fp8) latent_append_kernel<true, false><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
  else if (f32) latent_append_kernel<false, true><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
  else latent_append_kernel<false, false><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
  return check_launch(who);
}

extern "C" int pith_latent_gather(const pith_latent_gather_args* a, pith_stream_t stream) {
  const char* who = "pith_latent_gather";
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (a->B < 0 || a->rows < 0 || a->B > 0x7ffffffe || a->rows > 0x7fffffff - 4 * kGatherRows || a->table_width < 0 || a->table_width > 0x7fffffff)
    return fail(PITH_ERR_BAD_SHAPE, "%s: B = %lld, rows = %lld, table_width = %lld", who, (long long)a->B, (long long)a->rows, (long long)a->table_width);
  if (const int rc = check_cache(a->cache, who)) return rc;
  if (a->B == 0 || a->rows == 0) return PITH_OK;
  if (a->table_width == 0) return fail(PITH_ERR_BAD_SHAPE, "%s: an empty page table holds no rows", who);
  if (!a->page_table || !a->cu_rows || !a->latent_out || !a->k_pe_out) return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if ((a->B > 1 && a->table_rs < a->table_width) || (a->rows > 1 && (a->latent_rs < kLatent || a->k_pe_rs < kRope)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a row stride is shorter than a row", who);
  if (!aligned16(a->latent_out) || !aligned16(a->k_pe_out) || a->latent_rs % 8 || a->k_pe_rs % 8 || (uintptr_t)a->page_table % 4 || (uintptr_t)a->cu_rows % 4)
    return fail(PITH_ERR_MISALIGNED, "%s: outputs need 16-byte alignment", who);
  GatherParams p = {};
  p.cache = to_device(a->cache);
  p.table = a->page_table; p.cu_rows = a->cu_rows; p.latent_out = (__bf16*)a->latent_out; p.k_pe_out = (__bf16*)a->k_pe_out;
  p.table_rs = a->B > 1 ? a->table_rs : 0; p.latent_rs = a->latent_rs; p.k_pe_rs = a->k_pe_rs;
  p.B = (int)a->B; p.rows = (int)a->rows; p.table_width = (int)a->table_width;
  const int per_block = kWaves * kGatherRows;
  const dim3 grid((unsigned)((a->rows + per_block - 1) / per_block));
  begin_launch();
  if (a->cache.dtype == PITH_FP8_E4M3) latent_gather_kernel<true><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
  else latent_gather_kernel<false><<<grid, kThreads, 0, (hipStream_t)stream>>>(p);
  return check_launch(who);
}
