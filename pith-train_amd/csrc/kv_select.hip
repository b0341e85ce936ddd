// Which pages of a long cache a token attends to (include/pith_kv.h): a bound of q . k over every page from the least and largest values of its key
// features, then the pages with the largest bounds in the order of the sequence.
//
//   score(page) = max over the heads of the group of sum_d max(q_d least_d, q_d largest_d)
//
// A choice must not depend on the order of a sum, or the same scores would choose differently elsewhere: products of two bf16 values are exact in fp64, and
// their sum in it loses nothing that a rounding to fp32 would show. But only the pages around the last one chosen need that. So scores are formed by matrix
// instructions first, sum_d q+_d largest_d + q-_d least_d with q+ and q- the parts of q above and below zero, in fp32, beside the same sum of absolute values,
// S: 2 D terms, each addition off by at most 2^-23 of S, so that a page's score is off by at most E = 2^-14 S (twice what the additions can lose). The score v
// of the last one chosen by these is found by histograms of 256 equal parts of the range that it lies in, two most often, to within 2 E of an average page. The
// score of the last one that has to be chosen then lies above the least that a page from v on may have and below the most that one up to v may: a page that is above
// the latter with its E taken off is in, one below the former with its E added is out, and the few between are summed in fp64, if they are more than there are places.
// A page of another size is in question by itself alone. Infinities and NaN have no bound of the error: a page with one is summed in fp64 at once. NaN counts above all.
// Of equal scores all are in question. Up to 128 are ranked by comparing each with all; more by the bytes of their keys, a wave summing its own pages one after the
// other: 8 tokens over 2000 pages of one score 370 us, over 16000 2450 (18 and 70 where scores differ); one such token holds the call up.
// All of it is latency: 32 tokens with heads of 32 / 4 over up to 128 pages 12 us, one launch; 8 over up to 2048 pages 24 us, three launches with the
// bounds of the pages that the step filled: scores 10 (27 MB of bounds, 2.7 TB/s; four loads that wait for each other begin it), the choice 7 to 9 (1 until it knows what
// it is about, 0.5 for the scores, 2.3 for the histograms, 1.3 for the few pages in fp64, 1.6 to rank and write).
#include "cache_attn.h"
#include "kv_common.h"

#include <algorithm>
#include <type_traits>

namespace pith {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 128;  // pages of a workgroup that scores, sixteen a wave at a time

struct KVSelectParams {
  const __bf16 *q, *bounds;
  const int32_t *table, *lengths, *cu_q;
  int32_t *table_out, *lengths_out;
  uint2* pages_of;  // workspace, [tokens of the part * heads][row]: score and S of each page, then the keys of those in question
  int64_t q_ts, q_hs, table_rs, bounds_ps, row;
  int T, B, heads, group, pages, page_shift, table_width, keep, chunks, tokens;
  int first, last;  // the part's tokens
};

// A token and key-value head.
struct Item {
  int t, head, seq, length, end, visible, pages;  // end: of the sequence's tokens
  const int32_t* table;
};

__device__ __forceinline__ int pages_of(const KVSelectParams& p, int rows) { return (rows + (1 << p.page_shift) - 1) >> p.page_shift; }

__device__ __forceinline__ void see(const KVSelectParams& p, Item& x) {  // what token x.t sees of its sequence (a token that is nobody's: nothing)
  x.visible = !p.cu_q ? x.length : x.t < x.end ? min(max(x.length - x.end + x.t + 1, 0), x.length) : 0;
  x.pages = pages_of(p, x.visible);
}

__device__ __forceinline__ Item item_of(const KVSelectParams& p, int item, int lane) {
  Item x;
  x.t = item / p.heads;
  x.head = item - x.t * p.heads;
  if (!p.cu_q) {
    x.seq = x.t, x.end = x.t + 1, x.length = p.lengths[x.t];
  } else {  // 64 sequences at a time: the first that ends behind the token, whose length has come along
    x.seq = p.B - 1, x.end = 0, x.length = 0;  // (a token that is nobody's sees nothing: in front of the first offset, or behind all)
    int at_first = 0;
    asm("" : "+v"(at_first));  // (by a vector load, which is under way together with those below)
    const int first = p.cu_q[at_first];
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const int b = min(b0 + lane, p.B - 1), end = p.cu_q[b + 1], length = p.lengths[b];
      const uint64_t behind = __ballot(end > x.t);
      if (behind != 0) {
        const int i = __builtin_ctzll(behind);
        x.seq = min(b0 + i, p.B - 1), x.end = min(__builtin_amdgcn_readlane(end, i), p.T), x.length = __builtin_amdgcn_readlane(length, i);
        break;
      }
    }
    if (x.t < __builtin_amdgcn_readfirstlane(first)) x.end = 0, x.length = 0;
  }
  x.length = min(max(x.length, 0), p.table_width << p.page_shift);
  x.table = p.table + x.seq * p.table_rs;
  see(p, x);
  return x;
}

__device__ __forceinline__ uint32_t sort_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  return u >> 31 ? ~u : u | 0x80000000u;
}

typedef __attribute__((ext_vector_type(8))) short s16x8;

// The bounds of TILES times sixteen pages, `first` .. and so on, of which `held` exist: lane c + 16 g has eight features of page c, from 8 g on, of each 32.
template <int D, int TILES>
struct PageBounds {
  static constexpr int kSteps = D / 32;
  bf16x8 least[TILES][kSteps], largest[TILES][kSteps];

  __device__ __forceinline__ void load(const KVSelectParams& p, const Item& x, int first, int held, int lane) {
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int64_t page = safe_page(x.table[min(first + 16 * i + c, held - 1)], p.pages);
      const __bf16* const from = p.bounds + page * p.bounds_ps + (int64_t)x.head * (2 * D) + 8 * g;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        least[i][k] = *reinterpret_cast<const bf16x8*>(from + 32 * k);
        largest[i][k] = *reinterpret_cast<const bf16x8*>(from + D + 32 * k);
      }
    }
    // The split into q+ and q- asks for least <= largest; bounds of somebody else's making that are the other way round are exchanged. (As fp32 the upper of two
    // features is compared with the lower one behind it: that says too often at most.)
    int turned = 0;
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const u32x4 a = __builtin_bit_cast(u32x4, least[i][k]), b = __builtin_bit_cast(u32x4, largest[i][k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) turned |= (int)(__uint_as_float(a[e]) > __uint_as_float(b[e])) | (int)(bf16lo_to_f32(a[e]) > bf16lo_to_f32(b[e]));
      }
    if (__any(turned)) {
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const __bf16 a = least[i][k][e], b = largest[i][k][e];
            const bool other = (float)a > (float)b;
            least[i][k][e] = other ? b : a, largest[i][k][e] = other ? a : b;
          }
    }
  }

  // Scores and S (infinity: not known) of the token's head: lane c + 16 g has those of page c (whatever g). Operand A is sixteen heads, B sixteen pages, so a
  // lane's results are four heads of one page.
  __device__ __forceinline__ void score(const KVSelectParams& p, const Item& x, int lane, float2 (&out)[TILES]) const {
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < TILES; ++i) out[i] = make_float2(-INFINITY, 0.f);
#pragma unroll 1
    for (int h0 = 0; h0 < p.group; h0 += 16) {
      const __bf16* const from = p.q + x.t * p.q_ts + (int64_t)(x.head * p.group + min(h0 + c, p.group - 1)) * p.q_hs + 8 * g;
      s16x8 q[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) q[k] = *reinterpret_cast<const s16x8*>(from + 32 * k);
      f32x4 sum[TILES], mass[TILES];
#pragma unroll
      for (int i = 0; i < TILES; ++i) sum[i] = mass[i] = f32x4{};
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const s16x8 below = q[k] >> 15;  // all bits where q is below zero
        const auto bf = [](s16x8 v) __attribute__((always_inline)) { return __builtin_bit_cast(bf16x8, v); };
        const auto magnitude = [&](bf16x8 v) __attribute__((always_inline)) { return bf(__builtin_bit_cast(s16x8, v) & (short)0x7fff); };
        const bf16x8 up = bf(q[k] & ~below), down = bf(q[k] & below), down_size = magnitude(down);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          sum[i] = mfma16(up, largest[i][k], mfma16(down, least[i][k], sum[i]));
          mass[i] = mfma16(up, magnitude(largest[i][k]), mfma16(down_size, magnitude(least[i][k]), mass[i]));
        }
      }
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          out[i].x = fmaxf(out[i].x, sum[i][v]);
          out[i].y = fmaxf(out[i].y, mass[i][v] < INFINITY ? mass[i][v] : INFINITY);
        }
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) out[i] = make_float2(quad_max(out[i].x), quad_max(out[i].y));
  }
};

// A page's score in fp64, by a whole wavefront: eight lanes a head, eight heads at a time.
template <int D>
__device__ __forceinline__ float exact_score(const KVSelectParams& p, const Item& x, int index, int lane) {
  constexpr int E = D / 8;  // features of a lane
  const int64_t page = safe_page(x.table[index], p.pages);
  const __bf16* const from = p.bounds + page * p.bounds_ps + (int64_t)x.head * (2 * D) + E * (lane & 7);
  bf16x8 least[E / 8], largest[E / 8];
#pragma unroll
  for (int e = 0; e < E / 8; ++e) {
    least[e] = *reinterpret_cast<const bf16x8*>(from + 8 * e);
    largest[e] = *reinterpret_cast<const bf16x8*>(from + D + 8 * e);
  }
  float best = -INFINITY;
#pragma unroll 1
  for (int h0 = 0; h0 < p.group; h0 += 8) {
    const __bf16* const row = p.q + x.t * p.q_ts + (int64_t)(x.head * p.group + min(h0 + (lane >> 3), p.group - 1)) * p.q_hs + E * (lane & 7);
    double sum = 0.;
#pragma unroll
    for (int e = 0; e < E / 8; ++e) {
      const bf16x8 q = *reinterpret_cast<const bf16x8*>(row + 8 * e);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += __builtin_elementwise_maximum((double)q[k] * (double)least[e][k], (double)q[k] * (double)largest[e][k]);  // (NaN stays; in 32 bits they could overflow)
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) sum += __shfl_xor(sum, d);
    best = __builtin_elementwise_maximum(best, (float)sum);
  }
#pragma unroll
  for (int d = 8; d < 64; d <<= 1) best = __builtin_elementwise_maximum(best, __shfl_xor(best, d));
  return best;
}

// A workgroup: kChunk pages of a head, for p.tokens tokens, whose bounds are read once for all of a sequence.
template <int D>
__global__ __launch_bounds__(kThreads) void kv_score_kernel(KVSelectParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = blockIdx.x % p.chunks, part = blockIdx.x / p.chunks, t0 = p.first + part / p.heads * p.tokens, head = part % p.heads;
  const int first = chunk * kChunk + 32 * wave;
  PageBounds<D, 2> bounds;
  int loaded = -1;  // sequence
  Item x;
  x.end = 0;
#pragma unroll 1
  for (int t = t0; t < min(t0 + p.tokens, p.last); ++t) {
    const int item = t * p.heads + head;
    if (t < x.end) {
      x.t = t;
      see(p, x);
    } else {
      x = item_of(p, item, lane);
    }
    if (x.pages <= p.keep || first >= x.pages - 1) continue;  // (the token's own page is not scored)
    if (x.seq != loaded) bounds.load(p, x, first, pages_of(p, x.length), lane);
    loaded = x.seq;
    float2 found[2];
    bounds.score(p, x, lane, found);
    if (lane < 32) reinterpret_cast<float2*>(p.pages_of)[(item - p.first * p.heads) * p.row + first + lane] = lane < 16 ? found[0] : found[1];  // (of those behind the last: not read)
  }
}

// Sums and maxima over a workgroup, one barrier each (the other half of what is shared is still being read from the call before).
template <int THREADS, int E>
struct Team {
  static constexpr int kGroups = THREADS / 64, kListed = 128;
  struct Shared {
    int2 sums[2][kGroups];
    float4 survey[kGroups];
    __attribute__((aligned(16))) int histogram[2][256];
    __attribute__((aligned(16))) int chosen[E * kGroups];
    int listed;
    uint2 list[kListed];
  };
  Shared& shared;
  int turn;
  __device__ __forceinline__ explicit Team(Shared& s) : shared(s), turn(0) {}
  static __device__ __forceinline__ float wave_max(float x) { return quad_max(group_reduce<16>(x, [](float y, float z) { return fmaxf(y, z); })); }
  __device__ __forceinline__ float2 most(float a, float b) {
    a = wave_max(a), b = wave_max(b);
    if ((threadIdx.x & 63) == 63) shared.sums[turn][threadIdx.x >> 6] = make_int2(__float_as_int(a), __float_as_int(b));
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kGroups; ++w) {
      const int2 s = shared.sums[turn][w];
      a = fmaxf(a, __int_as_float(s.x)), b = fmaxf(b, __int_as_float(s.y));
    }
    turn ^= 1;
    return make_float2(a, b);
  }
  // Once: the largest a, b and c, and the sum of d (added in one order: of all threads the same).
  __device__ __forceinline__ float4 survey(float a, float b, float c, float d) {
    a = wave_max(a), b = wave_max(b), c = wave_max(c);
    d = quad_sum(group_reduce<16>(d, [](float y, float z) { return y + z; }));
    if ((threadIdx.x & 63) == 63) shared.survey[threadIdx.x >> 6] = make_float4(a, b, c, d);
    __syncthreads();
    d = 0.f;
#pragma unroll
    for (int w = 0; w < kGroups; ++w) {
      const float4 s = shared.survey[w];
      a = fmaxf(a, s.x), b = fmaxf(b, s.y), c = fmaxf(c, s.z), d += s.w;
    }
    return make_float4(a, b, c, d);
  }
  __device__ __forceinline__ int2 sums(int x, int y) {
    x = wave_scan(x), y = wave_scan(y);
    if ((threadIdx.x & 63) == 63) shared.sums[turn][threadIdx.x >> 6] = make_int2(x, y);
    __syncthreads();
    int2 all = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < kGroups; ++w) all.x += shared.sums[turn][w].x, all.y += shared.sums[turn][w].y;
    turn ^= 1;
    return all;
  }
};

// A score as the search for v sees it: infinities and what comes near them become large numbers, in the same order.
__device__ __forceinline__ float in_range(float x) { return x != x ? 1e37f : fminf(fmaxf(x, -1e37f), 1e37f); }

// How far a score of the matrix instructions may be off (S: the sum of the absolute values, infinity where the score is that of exact_score) and terms that are
// below the normal range.
__device__ __forceinline__ float error_of(float mass) { return (mass < INFINITY ? mass * 0x1p-14f : 0.f) + 0x1p-60f; }

// The part of a histogram, from the highest, in which the left-th lies; `left` becomes its rank in there. Every wave looks it up, four parts a lane.
__device__ __forceinline__ int part_with(const int* histogram, int lane, int& left) {
  const int4 h = *reinterpret_cast<const int4*>(&histogram[252 - 4 * lane]);
  const int mine = h.x + h.y + h.z + h.w, upto = wave_scan(mine);
  const int j = __builtin_ctzll(__ballot(upto >= left));
  left -= __builtin_amdgcn_readlane(upto - mine, j);
  const int hw = __builtin_amdgcn_readlane(h.w, j), hz = __builtin_amdgcn_readlane(h.z, j), hy = __builtin_amdgcn_readlane(h.y, j);
  int part = 255 - 4 * j;
  if (left > hw) {
    left -= hw, --part;
    if (left > hz) {
      left -= hz, --part;
      if (left > hy) left -= hy, --part;
    }
  }
  return part;
}

// Of the n pages of a token and head the `want` (fewer) with the largest scores: their numbers to out, in their order. score: in_range, of pages tid + THREADS e;
// error(e): how far each may be off; number(e): the table's entries of those; memory: room for n. By a whole workgroup.
template <int D, int THREADS, int E, typename F, typename N>
__device__ __forceinline__ void choose(const KVSelectParams& p, const Item& x, Team<THREADS, E>& team, const float (&score)[E], const F& error, const N& number, int n, int want, uint2* memory, int32_t* out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto& shared = team.shared;
  const auto each = [&](const auto& f) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (tid + THREADS * e < n) f(e, score[e]);
  };
  if (tid < 256) shared.histogram[0][tid] = 0;
  if (tid == 0) shared.listed = 0;
  float a = -INFINITY, b = -INFINITY, top = 0.f, sum = 0.f;
  const float share = 1.f / (float)n;
  each([&](int e, float s) __attribute__((always_inline)) { a = fmaxf(a, s), b = fmaxf(b, -s), top = fmaxf(top, error(e)), sum += error(e) * share; });
  const float4 about = team.survey(a, b, top, sum);
  float high = about.x, low = -about.y;  // v lies between
  const float worst = about.z, off = 2.f * about.w;  // the largest error, twice the mean: v need not be known better
  int left = want;  // v is the how many-th of those between them
  int turn = 0;
#pragma unroll 1
  for (; high - low > off; turn ^= 1) {
    const float scale = 255.f / (high - low);
    const auto part_of = [&](float s) __attribute__((always_inline)) { return min((int)((s - low) * scale), 255); };  // (low: 0, high: another)
    if (tid < 256) shared.histogram[turn ^ 1][tid] = 0;
    each([&](int, float s) __attribute__((always_inline)) {
      if (s >= low && s <= high) atomicAdd(&shared.histogram[turn][part_of(s)], 1);
    });
    __syncthreads();
    const int part = part_with(shared.histogram[turn], lane, left);
    a = b = -INFINITY;
    each([&](int, float s) __attribute__((always_inline)) {
      if (s >= low && s <= high && part_of(s) == part) a = fmaxf(a, s), b = fmaxf(b, -s);
    });
    const float2 r = team.most(a, b);
    high = r.x, low = -r.y;
  }

  // The score of the last one chosen, in fp64, lies between the least that any page from `low` on may have (`want` pages at least are there) and the most that any up to
  // `high` may (fewer than `want` are not among these). Where errors are much alike, the largest stands for all of them, which saves a barrier (0.4 us).
  int in = 0, open = 0;
  uint32_t is_in = 0, is_open = 0;  // bit e
  const auto sort_out = [&](int e, float s, float off, float least, float most) __attribute__((always_inline)) {
    const bool yes = s - off > most, no = s + off < least;
    in += yes, open += !yes && !no;
    is_in |= (uint32_t)yes << e, is_open |= (uint32_t)(!yes && !no) << e;
  };
  if (worst <= 2.f * off) {  // (uniform)
    each([&](int e, float s) __attribute__((always_inline)) { sort_out(e, s, worst, low - worst, high + worst); });
  } else {
    a = b = -INFINITY;
    each([&](int e, float s) __attribute__((always_inline)) {
      const float off = error(e);
      a = s >= low ? fmaxf(a, off - s) : a;
      b = s <= high ? fmaxf(b, s + off) : b;
    });
    const float2 r = team.most(a, b);
    each([&](int e, float s) __attribute__((always_inline)) { sort_out(e, s, error(e), -r.x, r.y); });
  }
  const int2 all = team.sums(in, open);
  const int places = want - all.x;  // for those in question
  // f(e, how many of those that `mine` says come before the thread's page e), in the pages' order: of all waves' counts four a lane, and their sums so far.
  const auto place = [&](const auto& mine, const auto& f) __attribute__((always_inline)) {
    constexpr int kWaves = THREADS / 64;
    static_assert(kWaves % 4 == 0 && E * kWaves <= 256, "four counts a lane");
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t bits = __ballot(mine(e));
      if (lane == 0) shared.chosen[e * kWaves + wave] = __popcll(bits);
    }
    __syncthreads();
    const int4 c = lane < E * kWaves / 4 ? *reinterpret_cast<const int4*>(&shared.chosen[4 * lane]) : make_int4(0, 0, 0, 0);
    const int four = c.x + c.y + c.z + c.w, nth = wave & 3;
    const int upto = wave_scan(four) - four + (nth > 0 ? c.x : 0) + (nth > 1 ? c.y : 0) + (nth > 2 ? c.z : 0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t bits = __ballot(mine(e));
      f(e, __builtin_amdgcn_readlane(upto, e * (kWaves / 4) + __builtin_amdgcn_readfirstlane(wave >> 2)) + __popcll(bits & ((1ull << lane) - 1)));
    }
  };
  if (all.y == places) {
    is_in |= is_open;
  } else if (all.y <= Team<THREADS, E>::kListed) {  // (uniform)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if ((is_open >> e) & 1) shared.list[atomicAdd(&shared.listed, 1)].x = tid + THREADS * e;  // (in any order: what follows goes by the pages' numbers)
    __syncthreads();
#pragma unroll 1
    for (int k = wave; k < all.y; k += THREADS / 64) {
      const float exact = exact_score<D>(p, x, __builtin_amdgcn_readfirstlane(shared.list[k].x), lane);
      if (lane == 0) shared.list[k].y = sort_key(exact);
    }
    __syncthreads();
    // a page in question is in if fewer than `places` of the others are in front of it
#pragma unroll 1
    for (int e = 0; e < E; ++e) {
      if (__any((is_open >> e) & 1)) {
        const uint32_t i = tid + THREADS * e;
        uint32_t key = 0;
        for (int k = 0; k < all.y; ++k) key = shared.list[k].x == i ? shared.list[k].y : key;
        int rank = 0;
        for (int k = 0; k < all.y; ++k) {
          const uint2 other = shared.list[k];
          rank += other.y > key || (other.y == key && other.x < i);
        }
        is_in |= (uint32_t)(((is_open >> e) & 1) && rank < places) << e;
      }
    }
  } else {
    // Many, equal ones most often: a wave sums its own pages, the key of the last one chosen is found by histograms of its bytes, and of those that have it the first are in.
#pragma unroll 1
    for (int e = 0; e < E; ++e) {
      uint64_t mine = __ballot((is_open >> e) & 1);
      while (mine != 0) {
        const int j = __builtin_ctzll(mine);
        mine &= mine - 1;
        const float exact = exact_score<D>(p, x, __builtin_amdgcn_readfirstlane(64 * wave + THREADS * e + j), lane);
        if (lane == j) memory[tid + THREADS * e].y = sort_key(exact);
      }
    }
    uint32_t border = 0;
    left = places;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      int* const histogram = shared.histogram[turn];
      __syncthreads();  // the round before has been read
      if (tid < 256) histogram[tid] = 0;
      __syncthreads();
#pragma unroll 1
      for (int e = 0; e < E; ++e)
        if ((is_open >> e) & 1) {
          const uint32_t key = memory[tid + THREADS * e].y;
          if (shift == 24 || (key ^ border) >> (shift + 8) == 0) atomicAdd(&histogram[(key >> shift) & 255], 1);
        }
      __syncthreads();
      border |= (uint32_t)part_with(histogram, lane, left) << shift;
    }
    uint32_t is_equal = 0;
#pragma unroll 1
    for (int e = 0; e < E; ++e)
      if ((is_open >> e) & 1) {
        const uint32_t key = memory[tid + THREADS * e].y;
        is_in |= (uint32_t)(key > border) << e, is_equal |= (uint32_t)(key == border) << e;
      }
    const auto equal = [&](int e) __attribute__((always_inline)) { return (is_equal >> e) & 1; };
    uint32_t first = 0;
    place(equal, [&](int e, int rank) __attribute__((always_inline)) { first |= (uint32_t)(rank < left) << e; });
    is_in |= is_equal & first;
    __syncthreads();  // the counts have been read
  }
  // their places
  const auto chosen = [&](int e) __attribute__((always_inline)) { return (is_in >> e) & 1; };
  place(chosen, [&](int e, int at) __attribute__((always_inline)) {
    if (chosen(e)) out[at] = number(e);
  });
}

// A page whose S is not known gets its score in fp64 (`index`: of lane 0's page; by a whole wavefront).
template <int D>
__device__ __forceinline__ float settle_unknown(const KVSelectParams& p, const Item& x, int index, bool real, float2 found, int lane) {
  float score = found.x;
  uint64_t unknown = __ballot(real && !(found.y < INFINITY));
  while (unknown != 0) {
    const int j = __builtin_ctzll(unknown);
    unknown &= unknown - 1;
    const float exact = exact_score<D>(p, x, __builtin_amdgcn_readfirstlane(index + j), lane);
    score = lane == j ? exact : score;
  }
  return in_range(score);
}

// What needs no scores: rows and places that stay empty, the token's own page, tokens that see no more pages than are kept. False: that was all.
__device__ __forceinline__ bool begin_choice(const KVSelectParams& p, const Item& x, int item, int32_t* out) {
  const int n = min(x.pages, p.keep);
  if (threadIdx.x == 0) p.lengths_out[item] = x.visible - ((x.pages - n) << p.page_shift);
  for (int i = n + threadIdx.x; i < p.keep; i += blockDim.x) out[i] = -1;
  if (x.pages <= p.keep) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) out[i] = x.table[i];
    return false;
  }
  if (threadIdx.x == 0) out[n - 1] = x.table[x.pages - 1];
  return n > 1;
}

template <int D, int THREADS, int E>
__global__ __launch_bounds__(THREADS) void kv_pick_kernel(KVSelectParams p) {
  __shared__ typename Team<THREADS, E>::Shared shared;
  const int item = p.first * p.heads + blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item x = item_of(p, item, lane);
  int32_t* const out = p.table_out + (int64_t)item * p.keep;
  if (!begin_choice(p, x, item, out)) return;
  uint2* const memory = p.pages_of + blockIdx.x * p.row;
  const int n = x.pages - 1;
  float score[E], s[E];
  constexpr bool kEarly = E <= 4;  // the table's entries come with the scores, and stay with the errors in registers (which do not hold 16 of each: read when they are wanted)
  int32_t early[kEarly ? E : 1];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if constexpr (kEarly) early[e] = x.table[min((int)threadIdx.x + THREADS * e, n - 1)];
    const float2 found = reinterpret_cast<const float2*>(memory)[min((int)threadIdx.x + THREADS * e, n - 1)];
    score[e] = found.x, s[e] = found.y;
  }
  bool known = true;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    known = known && s[e] < INFINITY;
    score[e] = known ? in_range(score[e]) : score[e];
  }
  if (__any(!known)) {  // (rare; by way of the memory, so that the loop has one body)
    float2* const mine = reinterpret_cast<float2*>(memory) + threadIdx.x;
#pragma unroll 1
    for (int e = 0; e < E; ++e) {
      const bool real = (int)threadIdx.x + THREADS * e < n;
      const float settled = settle_unknown<D>(p, x, 64 * wave + THREADS * e, real, real ? mine[THREADS * e] : make_float2(0.f, 0.f), lane);
      if (real) mine[THREADS * e].x = settled;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) score[e] = (int)threadIdx.x + THREADS * e < n ? mine[THREADS * e].x : 0.f;
  }
  Team<THREADS, E> team(shared);
  const auto error = [&](int e) __attribute__((always_inline)) {
    if constexpr (kEarly) return error_of(s[e]);
    else return error_of(reinterpret_cast<const float2*>(memory)[threadIdx.x + THREADS * e].y);
  };
  const auto number = [&](int e) __attribute__((always_inline)) {
    if constexpr (kEarly) return early[e];
    else return x.table[threadIdx.x + THREADS * e];
  };
  choose<D, THREADS, E>(p, x, team, score, error, number, n, p.keep - 1, memory, out);
}

// Scores and choice in one launch, for tables of up to kFewPages pages.
constexpr int kFewPages = 256, kSomePages = 2048, kMostPages = 16384;
template <int D>
__global__ __launch_bounds__(kThreads) void kv_pick_few_kernel(KVSelectParams p) {
  __shared__ typename Team<kThreads, 1>::Shared shared;
  __shared__ float2 scores[kFewPages];  // and how far they may be off
  const int item = p.first * p.heads + blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Item x = item_of(p, item, lane);
  int32_t* const out = p.table_out + (int64_t)item * p.keep;
  if (!begin_choice(p, x, item, out)) return;
  const int n = x.pages - 1;
  const int32_t number = x.table[min((int)threadIdx.x, n - 1)];
#pragma unroll 1
  for (int first = 32 * wave; first < n; first += kChunk) {
    float2 found[2];
    PageBounds<D, 2> bounds;
    bounds.load(p, x, first, n, lane);
    bounds.score(p, x, lane, found);
    const float2 mine = lane < 16 ? found[0] : found[1];
    const bool real = lane < 32 && first + lane < n;
    const float s = settle_unknown<D>(p, x, first, real, mine, lane);
    if (real) scores[first + lane] = make_float2(s, error_of(mine.y));
  }
  __syncthreads();
  const float score[1] = {scores[threadIdx.x].x}, error = scores[threadIdx.x].y;
  Team<kThreads, 1> team(shared);
  choose<D, kThreads, 1>(
      p, x, team, score, [&](int) __attribute__((always_inline)) { return error; }, [&](int) __attribute__((always_inline)) { return number; }, n, p.keep - 1, p.pages_of + blockIdx.x * p.row, out);
}

int check_select(const pith_kv_select_args* a, const char* who) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (const int rc = check_pages(a->pages, a->page_size, a->heads, a->dim, who)) return rc;
  if (const int rc = check_table(a->T, a->B, a->heads, a->table_width, a->page_size, !a->cu_q, who)) return rc;
  if (a->H < 1 || a->H > 1024 || a->H % a->heads) return fail(PITH_ERR_BAD_SHAPE, "%s: %lld query heads (at most 1024) of %lld key-value heads", who, (long long)a->H, (long long)a->heads);
  if (a->keep < 1 || a->keep > 1 << 20) return fail(PITH_ERR_BAD_SHAPE, "%s: keep = %lld pages (1 to 2^20)", who, (long long)a->keep);
  if (a->table_width > kMostPages) return fail(PITH_ERR_UNSUPPORTED, "%s: page tables of %lld pages, at most %d", who, (long long)a->table_width, kMostPages);
  if (a->T * a->heads > 0x7fffffff / ((a->table_width + kChunk - 1) / kChunk + 1) || a->T * a->heads > (int64_t)1 << 24)
    return fail(PITH_ERR_UNSUPPORTED, "%s: too many tokens for page tables of that width: call it with fewer at a time", who);
  return PITH_OK;
}

int64_t chunks_of(const pith_kv_select_args* a) { return (a->table_width + kChunk - 1) / kChunk; }

// Tokens are taken in parts of as many as 64 MB of scores serve (one at least), one behind the other: a prompt of 8192 tokens over 2048 pages, 4 heads, has 512 MB of them
// (2.91 ms in eight parts, 2.82 at once).
constexpr int64_t kPartBytes = 64 << 20;
int64_t part_of(const pith_kv_select_args* a) {
  const int64_t each = a->heads * chunks_of(a) * kChunk * (int64_t)sizeof(uint2);
  return std::max<int64_t>(std::min(a->T, each > 0 ? kPartBytes / each : a->T), 1);
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int64_t pith_kv_select_workspace_bytes(const pith_kv_select_args* a) {
  if (check_select(a, "pith_kv_select_workspace_bytes") != PITH_OK || a->B == 0) return 0;
  return a->T == 0 ? 0 : part_of(a) * a->heads * chunks_of(a) * kChunk * (int64_t)sizeof(uint2);
}

extern "C" int pith_kv_select(const pith_kv_select_args* a, pith_stream_t stream) {
  const char* who = "pith_kv_select";
  if (const int rc = check_select(a, who)) return rc;
  if (a->T == 0 || a->B == 0) return PITH_OK;
  if (a->table_width == 0) return fail(PITH_ERR_BAD_SHAPE, "%s: an empty page table holds no rows", who);
  if (!a->q || !a->bounds || !a->page_table || !a->lengths || !a->table_out || !a->lengths_out || !a->workspace)
    return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if ((a->B > 1 && a->table_rs < a->table_width) || (a->pages > 1 && a->bounds_ps < a->heads * 2 * a->dim) || (a->T > 1 && a->q_ts < a->dim) || (a->H > 1 && a->q_hs < a->dim))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a stride is shorter than what it steps over", who);
  if (!aligned16(a->q) || !aligned16(a->bounds) || (a->q_ts | a->q_hs) % 8 || (a->pages > 1 && a->bounds_ps % 8) || (uintptr_t)a->workspace % 256 ||
      (uintptr_t)a->page_table % 4 || (uintptr_t)a->lengths % 4 || (uintptr_t)a->cu_q % 4 || (uintptr_t)a->table_out % 4 || (uintptr_t)a->lengths_out % 4)
    return fail(PITH_ERR_MISALIGNED, "%s: q and bounds need 16-byte alignment and strides of multiples of 8, the workspace 256-byte alignment", who);
  const int64_t need = pith_kv_select_workspace_bytes(a);
  if (a->workspace_bytes < need) return fail(PITH_ERR_BAD_SHAPE, "%s: the workspace has %lld bytes, %lld are needed", who, (long long)a->workspace_bytes, (long long)need);
  KVSelectParams p = {};
  p.q = (const __bf16*)a->q; p.bounds = (const __bf16*)a->bounds; p.table = a->page_table; p.lengths = a->lengths; p.cu_q = a->cu_q;
  p.table_out = a->table_out; p.lengths_out = a->lengths_out; p.pages_of = (uint2*)a->workspace;
  p.q_ts = a->q_ts; p.q_hs = a->q_hs; p.table_rs = a->B > 1 ? a->table_rs : 0; p.bounds_ps = a->pages > 1 ? a->bounds_ps : 0;
  p.chunks = (int)chunks_of(a); p.row = (int64_t)p.chunks * kChunk;
  p.T = (int)a->T; p.B = (int)a->B; p.heads = (int)a->heads; p.group = (int)(a->H / a->heads);
  p.pages = (int)a->pages; p.page_shift = __builtin_ctzll((unsigned long long)a->page_size); p.table_width = (int)a->table_width; p.keep = (int)a->keep;
  hipStream_t s = (hipStream_t)stream;
  begin_launch();
  const auto launch = [&](auto d) {
    constexpr int D = decltype(d)::value;
    const int tokens = p.last - p.first;
    const unsigned items = (unsigned)(tokens * p.heads);
    if (a->table_width <= kFewPages) {
      kv_pick_few_kernel<D><<<items, kThreads, 0, s>>>(p);
      return;
    }
    if (a->keep > 1 && a->table_width > a->keep) {  // (else nothing is scored)
      // Tokens of a workgroup: those that a sequence has on average, up to four, as long as there are two workgroups for every compute unit. us of the whole call with
      // 1 / 2 / 4 / 8: 22 sequences of 7 over up to 674 pages, heads of 64 / 4, 53 / 46 / 44 / 46; 8 of 4 over up to 2048 39 / 33 / 31 / 31; 108 of 2 46 / 40 / 40 / 41.
      const int64_t each = (a->T + a->B - 1) / a->B, most = items * (int64_t)p.chunks / (2 * compute_units_or_default());
      p.tokens = (int)std::max<int64_t>(std::min<int64_t>({each, most, 4}), 1);
      kv_score_kernel<D><<<(unsigned)((tokens + p.tokens - 1) / p.tokens * p.heads * p.chunks), kThreads, 0, s>>>(p);
    }
    if (a->table_width <= kSomePages) kv_pick_kernel<D, 512, kSomePages / 512><<<items, 512, 0, s>>>(p);
    else kv_pick_kernel<D, 1024, kMostPages / 1024><<<items, 1024, 0, s>>>(p);
  };
  for (const int64_t part = part_of(a); p.first < p.T; p.first = p.last) {
    p.last = (int)std::min<int64_t>(p.first + part, p.T);
    if (a->dim == 128) launch(std::integral_constant<int, 128>());
    else launch(std::integral_constant<int, 64>());
  }
  return check_launch(who);
}
