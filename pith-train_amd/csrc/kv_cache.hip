// The key-value cache's rows: written as new tokens come (RMS norm and rotation of q and k, quantisation), and what the selection of pages wants to know of
// them, the least and largest value of every key feature of a page.
//
// Both move memory and little else. A row of a head is 16 bytes a lane: a group of dim / 8 lanes holds it in registers from the load to the store, its sums are a
// few steps between lanes, and the rotation's partner (half a row away) comes from the lane half a group away. Query, key and value rows are rows of
// one launch.
#include "cache_attn.h"
#include "kv_common.h"

#include <algorithm>

namespace pith {
namespace {

constexpr int kThreads = 256;
// From which on a wave takes a whole token. us with a wave a piece / a token, heads of 32 / 4, bf16: 256 tokens 8.3 / 8.2, 1024 8.8 / 9.4, 2048 12.0 / 10.7, 4096
// 20.3 / 15.2, 8192 44 / 36 (172 MB, 4.8 TB/s; a copy reaches 4.9); e4m3: 1024 9.2 / 10.0, 2048 13.4 / 11.6.
constexpr int64_t kManyTokens = 2048;

struct KVAppendParams {
  const __bf16 *q, *k, *v;
  const void *q_weight, *k_weight;
  const __bf16 *cos, *sin;
  const int64_t *pos, *slots;
  __bf16* q_out;
  int64_t P, rows;  // positions, slots
  int64_t q_ts, k_ts, v_ts, q_out_ts;
  int q_hs, k_hs, v_hs, q_out_hs;
  int T, H, per_wave;  // per_wave: pieces of a token's work for one wave
  float eps;
  KVCache cache;
};

__device__ __forceinline__ void unpack8(u32x4 x, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[2 * e] = bf16lo_to_f32(x[e]), v[2 * e + 1] = bf16hi_to_f32(x[e]);
}

// A wave takes a token, whose position and slot are then scalars, and of it `per_wave` pieces of 64 / (D / 8) heads each, those of q, then of k, then of v (the
// next one is on its way while one is computed): all of them where there are many tokens, so that the tables' rows and the weights come once, or one
// where there are few, and latency counts (kManyTokens).
// Weights: 0 none, 1 bf16, 2 fp32. The norm, the rotation and the division by the scale are fp32, rounded once (to nearest even; e4m3: the largest feature
// becomes +-448 exactly). The scale is the fp32 quotient, not a power of two, as in the latent cache.
template <int D, bool FP8, int WEIGHT>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KVAppendParams p) {
  constexpr int kLanes = D / 8, kHeads = 64 / kLanes;
  const int lane = threadIdx.x & 63, sub = lane % kLanes, group = lane / kLanes;
  const int heads = p.cache.heads, q_pieces = (p.H + kHeads - 1) / kHeads, kv_pieces = (heads + kHeads - 1) / kHeads, pieces = q_pieces + 2 * kv_pieces;
  const int wave = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (pieces + p.per_wave - 1) / p.per_wave;
  const int t = __builtin_amdgcn_readfirstlane(wave / waves);
  if (t >= p.T) return;
  const int first = (wave - t * waves) * p.per_wave, last = min(first + p.per_wave, pieces) - 1;
  const int64_t slot = p.slots[t];
  const bool kept = slot >= 0 && slot < p.rows;
  const int64_t at = clamped_position(p.pos[t], p.P) * D + 8 * sub;

  // What piece i is about: 0 q, 1 k, 2 v; its first head.
  const auto what_of = [&](int i, int& head0) __attribute__((always_inline)) {
    const int what = i < q_pieces ? 0 : i < q_pieces + kv_pieces ? 1 : 2;
    head0 = (i - (what == 0 ? 0 : what == 1 ? q_pieces : q_pieces + kv_pieces)) * kHeads;
    return what;
  };
  const auto load = [&](int i) __attribute__((always_inline)) {
    int head0;
    const int what = what_of(i, head0);
    const __bf16* const base = what == 0 ? p.q + t * p.q_ts : what == 1 ? p.k + t * p.k_ts : p.v + t * p.v_ts;
    const int hs = what == 0 ? p.q_hs : what == 1 ? p.k_hs : p.v_hs, head = min(head0 + group, (what == 0 ? p.H : heads) - 1);
    return *reinterpret_cast<const u32x4*>(base + (head * hs + 8 * sub));
  };
  u32x4 next = load(first);
  float c[8], s[8], qw[8], kw[8];
  unpack8(*reinterpret_cast<const u32x4*>(p.cos + at), c);
  unpack8(*reinterpret_cast<const u32x4*>(p.sin + at), s);
  const auto weights = [&](const void* from, float (&w)[8]) __attribute__((always_inline)) {
    if constexpr (WEIGHT == 2) {
      const f32x4* const x = reinterpret_cast<const f32x4*>(from) + 2 * sub;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = x[e >> 2][e & 3];
    } else if constexpr (WEIGHT == 1) {
      unpack8(reinterpret_cast<const u32x4*>(from)[sub], w);
    }
  };
  weights(p.q_weight, qw);
  weights(p.k_weight, kw);
  const float sign = sub >= kLanes / 2 ? 1.f : -1.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] *= sign;

#pragma unroll 1
  for (int i = first; i <= last; ++i) {
    float x[8];
    unpack8(next, x);
    next = load(min(i + 1, last));
    int head0;
    const int what = what_of(i, head0), head = head0 + group;
    if (what != 0 && !kept) break;  // (k and v are the last)
    if (what != 2) {
      if constexpr (WEIGHT != 0) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += x[e] * x[e];
        const float inv = rsqrtf(group_reduce<kLanes>(sum, [](float a, float b) { return a + b; }) * (1.f / D) + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (what == 0 ? qw[e] : kw[e]);
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[e] * c[e] + other_half<kLanes>(x[e]) * s[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = y[e];
    }
    const auto packed = [&]() __attribute__((always_inline)) {
      u32x4 out;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
      return out;
    };
    if (what == 0) {
      if (head < p.H) *reinterpret_cast<u32x4*>(p.q_out + t * p.q_out_ts + (head * p.q_out_hs + 8 * sub)) = packed();
      continue;
    }
    const int64_t page = slot >> p.cache.page_shift, in_page = ((int64_t)head << p.cache.page_shift) + (slot & ((1 << p.cache.page_shift) - 1));
    char* const dst = what == 1 ? p.cache.k + page * p.cache.k_ps : p.cache.v + page * p.cache.v_ps;
    if constexpr (FP8) {
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
      const float scale = group_reduce<kLanes>(top, [](float a, float b) { return fmaxf(a, b); }) / kFp8Max;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = scale > 0.f ? x[e] / scale : x[e];  // (a row of zeros stays one; NaN stays NaN)
        y[e] = z > kFp8Max ? kFp8Max : (z < -kFp8Max ? -kFp8Max : z);
      }
      u32x2 out;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * e], y[4 * e + 1], 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * e + 2], y[4 * e + 3], word, true);
        out[e] = (uint32_t)word;
      }
      if (head < heads) {
        *reinterpret_cast<u32x2*>(dst + in_page * D + 8 * sub) = out;
        if (sub == 0) {
          if (what == 1) p.cache.k_scale[page * p.cache.k_scale_ps + in_page] = scale;
          else p.cache.v_scale[page * p.cache.v_scale_ps + in_page] = scale;
        }
      }
    } else {
      if (head < heads) *reinterpret_cast<u32x4*>(dst + in_page * (2 * D) + 16 * sub) = packed();
    }
  }
}

struct KVBoundsParams {
  KVCache cache;
  __bf16* bounds;
  const int32_t *table, *lengths, *cu_q;
  int64_t table_rs, bounds_ps;
  int T, table_width;
};

// The least and largest of rows with a NaN are NaN.
__device__ __forceinline__ float least(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float largest(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Pages first .. last - 1 of sequence b that its new tokens filled. Token offsets count as their maximum so far, from 0 to T, so that whatever they hold no token belongs
// to two sequences: the largest of the first b + 1, by a whole wavefront, 256 of them at a time, and more than that only if those and the sequence's own two do not say already
// that there is no page (they can only say too many).
struct Filled {
  int first, last;
};
__device__ __forceinline__ Filled filled_pages(const KVBoundsParams& p, int b, int lane) {
  const int shift = p.cache.page_shift;
  const auto pages = [&](int cached, int n) __attribute__((always_inline)) {
    const int length = min(max(cached, 0), p.table_width << shift);
    return Filled{max(length - n, 0) >> shift, length >> shift};
  };
  if (!p.cu_q) return pages(p.lengths[b], 1);
  const auto load = [&](int i0, int (&x)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = p.cu_q[min(i0 + 64 * k + lane, b)];
  };
  int x[4], end = p.cu_q[b + 1], most = p.cu_q[b], cached = p.lengths[b];
  load(0, x);
  asm volatile("" : "+s"(end), "+s"(most), "+s"(cached), "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));  // one wait for all of them, not one each where they are used
  const auto by = [&](int most_) __attribute__((always_inline)) {
    const int begin = __builtin_amdgcn_readlane(wave_scan_max(max(max(max(x[0], x[1]), max(x[2], x[3])), max(most_, 0))), 63);
    return pages(cached, max(min(max(end, 0), p.T) - min(begin, p.T), 0));
  };
  Filled f = by(most);
  if (b >= 256 && f.first < f.last) {
    int more = max(max(x[0], x[1]), max(x[2], x[3]));
    for (int i0 = 256; i0 <= b; i0 += 256) {
      load(i0, x);
      more = max(more, max(max(x[0], x[1]), max(x[2], x[3])));
    }
    f = by(more);
  }
  return f;
}

// blockIdx.x: sequence, blockIdx.y: key-value head, blockIdx.z: every how many-th of the pages that its new tokens filled. A group of lanes takes every
// 256 / kLanes-th row; what the groups found meets in LDS.
template <int D, bool FP8>
__global__ __launch_bounds__(kThreads) void kv_bounds_kernel(KVBoundsParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  __shared__ float found[2][kGroups][D];
  const int sub = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int b = blockIdx.x, head = blockIdx.y;
  const int page_size = 1 << p.cache.page_shift;
  const Filled filled = filled_pages(p, b, threadIdx.x & 63);
  for (int i = filled.first + blockIdx.z; i < filled.last; i += gridDim.z) {
    const int64_t page = safe_page(p.table[b * p.table_rs + i], p.cache.pages);
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
    const char* const rows = p.cache.k + page * p.cache.k_ps + (int64_t)head * page_size * (FP8 ? D : 2 * D);
    constexpr int kAtOnce = 4;  // rows in flight (those behind the page's last: that one again)
    for (int r0 = group; r0 < page_size; r0 += kAtOnce * kGroups) {
      u32x4 raw[kAtOnce];
      float scale[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int r = min(r0 + k * kGroups, page_size - 1);
        if constexpr (FP8) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(rows + (int64_t)r * D + 8 * sub);
          raw[k][0] = x[0], raw[k][1] = x[1];
          scale[k] = p.cache.k_scale[page * p.cache.k_scale_ps + (int64_t)head * page_size + r];
        } else {
          raw[k] = *reinterpret_cast<const u32x4*>(rows + (int64_t)r * (2 * D) + 16 * sub);
        }
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        float x[8];
        if constexpr (FP8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bf16x2 two = (e & 1) ? fp8x2_to_bf16<true>(raw[k][e >> 1]) : fp8x2_to_bf16<false>(raw[k][e >> 1]);
            x[2 * e] = (float)two[0] * scale[k], x[2 * e + 1] = (float)two[1] * scale[k];
          }
        } else {
          unpack8(raw[k], x);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] = least(lo[e], x[e]), hi[e] = largest(hi[e], x[e]);
      }
    }
    __syncthreads();  // the page before has been read
#pragma unroll
    for (int e = 0; e < 8; ++e) found[0][group][8 * sub + e] = lo[e], found[1][group][8 * sub + e] = hi[e];
    __syncthreads();
    if (threadIdx.x < 2 * D) {
      const int which = threadIdx.x / D, d = threadIdx.x % D;
      float x = found[which][0][d];
      for (int g = 1; g < kGroups; ++g) x = which == 0 ? least(x, found[0][g][d]) : largest(x, found[1][g][d]);
      p.bounds[page * p.bounds_ps + (int64_t)head * (2 * D) + threadIdx.x] = (__bf16)x;
    }
  }
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int pith_kv_append(const pith_kv_append_args* a, pith_stream_t stream) {
  const char* who = "pith_kv_append";
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (const int rc = check_cache(a->cache, who)) return rc;
  const int64_t dim = a->cache.dim, heads = a->cache.heads;
  if (a->T < 0 || a->T > 0x7fffffff || a->P < 1 || a->H < 1 || a->H > 1024)
    return fail(PITH_ERR_BAD_SHAPE, "%s: T = %lld tokens, %lld query heads (1 to 1024), tables of %lld positions", who, (long long)a->T, (long long)a->H, (long long)a->P);
  if (a->T == 0) return PITH_OK;
  if (a->T * (a->H + 2 * heads) > 0x7fffffff - 64) return fail(PITH_ERR_UNSUPPORTED, "%s: 2^31 rows or more in a call", who);
  const int64_t far = 0x3fffffff;  // offsets within a token are counted in 32 bits
  if (a->H * a->q_hs > far || a->H * a->q_out_hs > far || heads * a->k_hs > far || heads * a->v_hs > far)
    return fail(PITH_ERR_UNSUPPORTED, "%s: heads of a token that lie 2^30 elements apart", who);
  if (!a->q || !a->k || !a->v || !a->q_out || !a->cos || !a->sin || !a->position_ids || !a->slots || (a->q_weight == nullptr) != (a->k_weight == nullptr))
    return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL (the weights are given together or not at all)", who);
  if (a->q_weight && a->weight_dtype != PITH_BF16 && a->weight_dtype != PITH_F32) return fail(PITH_ERR_BAD_DTYPE, "%s: weight_dtype %d", who, a->weight_dtype);
  if ((a->T > 1 && (a->q_ts < dim || a->k_ts < dim || a->v_ts < dim || a->q_out_ts < dim)) || (a->H > 1 && (a->q_hs < dim || a->q_out_hs < dim)) ||
      (heads > 1 && (a->k_hs < dim || a->v_hs < dim)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a stride is shorter than a row", who);
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->q_out) || !aligned16(a->cos) || !aligned16(a->sin) || !aligned16(a->q_weight) ||
      !aligned16(a->k_weight) || (a->q_ts | a->q_hs | a->k_ts | a->k_hs | a->v_ts | a->v_hs | a->q_out_ts | a->q_out_hs) % 8 || (uintptr_t)a->position_ids % 8 ||
      (uintptr_t)a->slots % 8)
    return fail(PITH_ERR_MISALIGNED, "%s: q, k, v, q_out, weights and tables need 16-byte alignment and strides of multiples of 8", who);
  KVAppendParams p = {};
  p.q = (const __bf16*)a->q; p.k = (const __bf16*)a->k; p.v = (const __bf16*)a->v; p.q_out = (__bf16*)a->q_out;
  p.q_weight = a->q_weight; p.k_weight = a->k_weight; p.cos = (const __bf16*)a->cos; p.sin = (const __bf16*)a->sin;
  p.pos = a->position_ids; p.slots = a->slots; p.P = a->P; p.rows = a->cache.pages * a->cache.page_size;
  p.q_ts = a->q_ts; p.k_ts = a->k_ts; p.v_ts = a->v_ts; p.q_out_ts = a->q_out_ts;
  p.q_hs = (int)a->q_hs; p.k_hs = (int)a->k_hs; p.v_hs = (int)a->v_hs; p.q_out_hs = (int)a->q_out_hs;
  p.T = (int)a->T; p.H = (int)a->H; p.eps = a->eps;
  p.cache = to_device(a->cache);
  const int64_t per_piece = 512 / dim, pieces = (a->H + per_piece - 1) / per_piece + 2 * ((heads + per_piece - 1) / per_piece);
  p.per_wave = a->T >= kManyTokens ? (int)pieces : 1;
  const int64_t waves = a->T * ((pieces + p.per_wave - 1) / p.per_wave);
  const unsigned grid = (unsigned)((waves + kThreads / 64 - 1) / (kThreads / 64));
  hipStream_t s = (hipStream_t)stream;
  begin_launch();
  const bool fp8 = a->cache.dtype == PITH_FP8_E4M3;
  const int weight = !a->q_weight ? 0 : a->weight_dtype == PITH_BF16 ? 1 : 2;
  const auto launch = [&](auto d, auto f) {
    constexpr int D = decltype(d)::value;
    constexpr bool F = decltype(f)::value;
    if (weight == 0) kv_append_kernel<D, F, 0><<<grid, kThreads, 0, s>>>(p);
    else if (weight == 1) kv_append_kernel<D, F, 1><<<grid, kThreads, 0, s>>>(p);
    else kv_append_kernel<D, F, 2><<<grid, kThreads, 0, s>>>(p);
  };
  using std::integral_constant;
  if (dim == 128 && fp8) launch(integral_constant<int, 128>(), integral_constant<bool, true>());
  else if (dim == 128) launch(integral_constant<int, 128>(), integral_constant<bool, false>());
  else if (fp8) launch(integral_constant<int, 64>(), integral_constant<bool, true>());
  else launch(integral_constant<int, 64>(), integral_constant<bool, false>());
  return check_launch(who);
}

extern "C" int pith_kv_bounds(const pith_kv_bounds_args* a, pith_stream_t stream) {
  const char* who = "pith_kv_bounds";
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (const int rc = check_cache(a->cache, who)) return rc;
  const pith_kv_cache& c = a->cache;
  if (const int rc = check_table(a->T, a->B, c.heads, a->table_width, c.page_size, !a->cu_q, who)) return rc;
  if (a->T == 0 || a->B == 0) return PITH_OK;
  if (a->table_width == 0) return fail(PITH_ERR_BAD_SHAPE, "%s: an empty page table holds no rows", who);
  if (!a->bounds || !a->page_table || !a->lengths) return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if ((a->B > 1 && a->table_rs < a->table_width) || (c.pages > 1 && a->bounds_ps < c.heads * 2 * c.dim))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a stride is shorter than what it steps over", who);
  if (!aligned16(a->bounds) || (c.pages > 1 && a->bounds_ps % 8) || (uintptr_t)a->page_table % 4 || (uintptr_t)a->lengths % 4 || (uintptr_t)a->cu_q % 4)
    return fail(PITH_ERR_MISALIGNED, "%s: bounds need 16-byte alignment and a page stride of a multiple of 8", who);
  KVBoundsParams p = {};
  p.cache = to_device(c);
  p.bounds = (__bf16*)a->bounds; p.table = a->page_table; p.lengths = a->lengths; p.cu_q = a->cu_q;
  p.table_rs = a->B > 1 ? a->table_rs : 0; p.bounds_ps = c.pages > 1 ? a->bounds_ps : 0;
  p.T = (int)a->T; p.table_width = (int)a->table_width;
  const int64_t most = a->T / c.page_size + 1;  // pages that the tokens of one sequence can fill
  // Workgroups of a sequence and head, which share its pages: up to 64 where there are few of them, 8 where they are thousands, one each of which could be a prompt (us of a
  // decoding step over heads of 128, 4 of them, 1024 sequences, with 17 / 8 19 / 10, 4096 with 64 / 8 262 / 36).
  const int64_t z = std::max<int64_t>(4096 / (a->B * c.heads), 8);
  const dim3 grid((unsigned)a->B, (unsigned)c.heads, (unsigned)std::min<int64_t>({most, z, 64}));
  hipStream_t s = (hipStream_t)stream;
  begin_launch();
  const bool fp8 = c.dtype == PITH_FP8_E4M3;
  if (c.dim == 128 && fp8) kv_bounds_kernel<128, true><<<grid, kThreads, 0, s>>>(p);
  else if (c.dim == 128) kv_bounds_kernel<128, false><<<grid, kThreads, 0, s>>>(p);
  else if (fp8) kv_bounds_kernel<64, true><<<grid, kThreads, 0, s>>>(p);
  else kv_bounds_kernel<64, false><<<grid, kThreads, 0, s>>>(p);
  return check_launch(who);
}
