// The products around the absorbed attention: q_nope W_uk into the latent space (with the rotation of q_pe), and W_uv o_latent out of it.
//
// Per head a [T x 128] x [128 x 512] product either way. With few tokens (a decoding step) it is the 4 MB of weights of 16 heads that have to come in,
// with many the queries and results, 1.5 KB a token and head, against 131 kflop: memory in both cases. So a wave takes a share of the output
// features, holds its part of the head's weights in registers as MFMA A operands (each weight is read once per workgroup), and walks the tokens,
// 16 at a time as the B operand (16x16x32: lane = token lane % 16, contraction 8 (lane / 16) + e), through a ring of LDS tiles with all but one in
// flight. The result tile then has the token as its column and consecutive features in a lane's registers, so rows leave straight from there.
// 128 heads, 512 tokens (100 MB, 21 us as a copy): 22 + 7 us the queries, 25 us the results; 16 heads, 32 tokens: 3.7 and 3.6 us.
#include "attn_tiles.h"
#include "latent_common.h"

namespace pith {
namespace {

struct AbsorbParams {
  const __bf16* x;
  const __bf16* weight;
  __bf16* out;
  __bf16* q_pe;
  const __bf16* cos;
  const __bf16* sin;
  const int64_t* pos;
  int64_t x_ts, x_hs, out_ts, out_hs, q_pe_ts, q_pe_hs, P;
  int T, H, tokens_per_block;
};

// kPairs pairs of q_pe a thread, THREADS / 32 rows (token * H + head) apart, workgroup n's from row n kPairs THREADS / 32 on. Their loads stand side by
// side: position, then its row of the tables, is one latency behind the other.
constexpr int kPairs = 4;

template <int THREADS>
__device__ __forceinline__ void rotate_queries(const AbsorbParams& p, int group) {
  const int rows = p.T * p.H, first = group * (kPairs * THREADS / 32) + (threadIdx.x >> 5), j = threadIdx.x & 31;
  uint32_t pair[kPairs];
  int64_t at[kPairs];
  __bf16* dst[kPairs];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    const int row = min(first + k * (THREADS / 32), rows - 1), t = row / p.H, h = row - t * p.H;
    at[k] = clamped_position(p.pos[t], p.P) * kRope;
    pair[k] = *reinterpret_cast<const uint32_t*>(p.x + t * p.x_ts + h * p.x_hs + kNope + 2 * j);
    dst[k] = p.q_pe + t * p.q_pe_ts + h * p.q_pe_hs;
  }
  float a[kPairs], b[kPairs];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) rotate_pair(pair[k], p.cos + at[k], p.sin + at[k], j, a[k], b[k]);
#pragma unroll
  for (int k = 0; k < kPairs; ++k)
    if (first + k * (THREADS / 32) < rows) {
      dst[k][j] = (__bf16)a[k];
      dst[k][kRope / 2 + j] = (__bf16)b[k];
    }
}

constexpr int kRotateThreads = 256;
__global__ __launch_bounds__(kRotateThreads) void absorb_rotate_kernel(AbsorbParams p) {
  rotate_queries<kRotateThreads>(p, blockIdx.x);
}

// The first `products` workgroups: q_latent features [64 WAVES x, + 64 WAVES) of a head, a block of tokens; the others (WAVES = 2) rotate. W_uk's rows are the
// contraction (d), so its fragments come transposed out of LDS, where it lies in slices of 128 features, 256 bytes a row; wave w's 64 features are four
// products whose rows are dealt so that a lane's results of two are eight consecutive features (product n, row 4 g + v: feature
// 32 (n / 2) + 8 g + 4 (n % 2) + v). Then the ring of tiles of 32 tokens takes that place. Fetched as fragments, queries took the address unit 64
// cycles a piece: 128 heads, 2048 tokens 215 us.
// Where several workgroups read a block's queries (WAVES = 2) they lie 8 apart: one XCD's cache serves them.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void absorb_query_kernel(AbsorbParams p, int products, int blocks) {
  constexpr int kSlices = WAVES / 2, kColumns = 8 / WAVES;  // of 128 features; workgroups to a head's block
  constexpr int kTokens = 32, kTile = kTokens * kRowBytes128, kRing = kSlices * 128 * kRowBytes128 / kTile + 1, kLoads = kTokens / 4 / WAVES;
  __shared__ __attribute__((aligned(1024))) char lds[kRing * kTile];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (WAVES == 2) {
    if ((int)blockIdx.x >= products) return rotate_queries<64 * WAVES>(p, blockIdx.x - products);
  }
  const int of = blockIdx.x / (8 * kColumns) * 8 + (blockIdx.x & 7), x = (blockIdx.x >> 3) % kColumns;  // head and block, column
  const int h = __builtin_amdgcn_readfirstlane(of / blocks);
  if (h >= p.H) return;
  const int t0 = (of - h * blocks) * p.tokens_per_block, t1 = min(t0 + p.tokens_per_block, p.T);
  const int tiles = (t1 - t0 + kTokens - 1) / kTokens;
  const int c = lane & 15, g = lane >> 4;
  const int first = 64 * (WAVES * x + wave);  // of the wave's features
  const auto request = [&](int i, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int region = kLoads * wave + k, r = 4 * region + (lane >> 4);
      load_lds16_at(p.x + (int64_t)min(t0 + kTokens * i + r, t1 - 1) * p.x_ts + h * p.x_hs + 8 * ((lane & 15) ^ row_swizzle(r)), lds + slot * kTile + 1024 * region);
    }
  };
  {
    const char* const weight = reinterpret_cast<const char*>(p.weight + (int64_t)h * (kNope + kValue) * kLatent + 64 * WAVES * x);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int region = 16 * wave + k, slice = region >> 5, r = 4 * (region & 31);  // (two waves fetch a slice)
      load_lds16(weight + r * 2 * kLatent + 256 * slice, (lane >> 4) * 2 * kLatent + 16 * ((lane & 15) ^ tile_swizzle(r + (lane >> 4))), lds + 1024 * region);
    }
  }
  request(0, kRing - 1);
  wait_loads<kLoads>();
  __syncthreads();
  bf16x8 w[4][4];
  const char* const slice = lds + (wave >> 1) * 128 * kRowBytes128;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      // lane 4 i + k of a 16-lane group brings four features of row i: group k of the product's 16
      const int feature = 64 * (wave & 1) + 32 * (n >> 1) + 8 * (c & 3) + 4 * (n & 1);
      const int row = 32 * st + 8 * g + (c >> 2);
      const char* lo = slice + swizzled_offset(row, feature >> 3) + ((feature & 7) << 1);
      const char* hi = slice + swizzled_offset(row + 4, feature >> 3) + ((feature & 7) << 1);
      w[n][st] = lds_read_transposed_at(lo, hi);
    }
  __syncthreads();
  for (int i = 1; i < min(tiles, kRing - 1); ++i) request(i, i - 1);
  int slot = kRing - 1;
  for (int i = 0; i < tiles; ++i) {
    if (i + kRing - 1 <= tiles) wait_loads<(kRing - 2) * kLoads>();
    else wait_loads<0>();
    __syncthreads();
    const char* const tile = lds + slot * kTile;
    if (i + kRing - 1 < tiles) request(i + kRing - 1, slot == 0 ? kRing - 1 : slot - 1);
    slot = slot + 1 == kRing ? 0 : slot + 1;
#pragma unroll
    for (int half = 0; half < kTokens / 16; ++half) {
      f32x4 acc[4] = {};
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const bf16x8 q = *reinterpret_cast<const bf16x8*>(tile + (16 * half + c) * kRowBytes128 + (((4 * st + g) ^ row_swizzle(c)) << 4));
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n] = mfma16(w[n][st], q, acc[n]);
      }
      const int t = t0 + kTokens * i + 16 * half + c;
      if (t < t1) {
        __bf16* const dst = p.out + (int64_t)t * p.out_ts + h * p.out_hs + first + 8 * g;
#pragma unroll
        for (int n = 0; n < 4; n += 2)
          *reinterpret_cast<u32x4*>(dst + 16 * n) = u32x4{pack_bf16x2(acc[n][0], acc[n][1]), pack_bf16x2(acc[n][2], acc[n][3]),
                                                         pack_bf16x2(acc[n + 1][0], acc[n + 1][1]), pack_bf16x2(acc[n + 1][2], acc[n + 1][3])};
      }
    }
  }
}

// o features [16 WAVES x, + 16 WAVES) of head y, tokens of block z. Rows of W_uv and of o_latent are both contiguous along the contraction, 1 KB each, but a
// fragment touches sixteen of them, which the address unit serves at a lane a cycle: so both come through LDS, a row an instruction. Wave w fetches its
// sixteen rows of weights into registers (64) by way of slot w of the ring, which then takes tiles of sixteen tokens, as many in flight as it has slots.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void absorb_value_kernel(AbsorbParams p) {
  constexpr int kRing = WAVES + 1, kTile = 16 * 2 * kLatent, kRows = 16 / WAVES;  // rows of a tile that a wave fetches
  __shared__ __attribute__((aligned(1024))) char lds[kRing * kTile];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y;
  const int t0 = blockIdx.z * p.tokens_per_block, t1 = min(t0 + p.tokens_per_block, p.T);
  const int tiles = (t1 - t0 + 15) >> 4;
  const int c = lane & 15, g = lane >> 4;
  const int first = 16 * (WAVES * blockIdx.x + wave);  // of the wave's features
  const auto row = [&](const __bf16* src, char* tile, int r) __attribute__((always_inline)) {
    load_lds16(reinterpret_cast<const char*>(src), (16 * lane) ^ (16 * row_swizzle(r)), tile + r * 2 * kLatent);
  };
  const auto request = [&](int i, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int r = kRows * wave + k;
      row(p.x + (int64_t)min(t0 + 16 * i + r, t1 - 1) * p.x_ts + h * p.x_hs, lds + slot * kTile, r);
    }
  };
  const auto fragment = [&](const char* tile, int st) __attribute__((always_inline)) {
    const uint32_t at = lds_address(tile) + c * 2 * kLatent + ((g ^ row_swizzle(c)) << 4);
    return *lds_at<bf16x8>((at ^ (64 * (st & 3))) + 256 * (st >> 2));
  };
#pragma unroll
  for (int r = 0; r < 16; ++r) row(p.weight + ((int64_t)h * (kNope + kValue) + kNope + first + r) * kLatent, lds + wave * kTile, r);
  request(0, WAVES);
  wait_loads<kRows>();
  bf16x8 w[16];
#pragma unroll
  for (int st = 0; st < 16; ++st) w[st] = fragment(lds + wave * kTile, st);
  __syncthreads();
  for (int i = 1; i < min(tiles, kRing - 1); ++i) request(i, i - 1);
  int slot = WAVES;
  for (int i = 0; i < tiles; ++i) {
    if (i + kRing - 1 <= tiles) wait_loads<(kRing - 2) * kRows>();
    else wait_loads<0>();
    __syncthreads();
    const char* const tile = lds + slot * kTile;
    if (i + kRing - 1 < tiles) request(i + kRing - 1, slot == 0 ? kRing - 1 : slot - 1);
    slot = slot + 1 == kRing ? 0 : slot + 1;
    f32x4 acc[2] = {};  // even and odd steps: two chains
#pragma unroll
    for (int st = 0; st < 16; ++st) acc[st & 1] = mfma16(w[st], fragment(tile, st), acc[st & 1]);
    acc[0] += acc[1];
    const int t = t0 + 16 * i + c;
    if (t < t1)
      *reinterpret_cast<u32x2*>(p.out + (int64_t)t * p.out_ts + h * p.out_hs + first + 4 * g) = u32x2{pack_bf16x2(acc[0][0], acc[0][1]), pack_bf16x2(acc[0][2], acc[0][3])};
  }
}

int check_absorb(const pith_latent_absorb_args* a, const char* who, int in_dim, int out_dim, AbsorbParams& p) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (a->T < 0 || a->T > 1 << 20 || a->H < 1 || a->H > 1024) return fail(PITH_ERR_BAD_SHAPE, "%s: T = %lld tokens, H = %lld heads (at most 2^20, 1024)", who, (long long)a->T, (long long)a->H);
  if (a->T * a->H > 1 << 28) return fail(PITH_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads: more than 2^28 rows", who, (long long)a->T, (long long)a->H);
  if (a->T == 0) return PITH_OK;
  if (!a->x || !a->weight || !a->out) return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if ((a->T > 1 && (a->x_ts < in_dim || a->out_ts < out_dim)) || (a->H > 1 && (a->x_hs < in_dim || a->out_hs < out_dim)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a stride is shorter than %d or %d features", who, in_dim, out_dim);
  if (!aligned16(a->x) || !aligned16(a->weight) || !aligned16(a->out) || (a->x_ts | a->x_hs | a->out_ts | a->out_hs) % 8)
    return fail(PITH_ERR_MISALIGNED, "%s: pointers need 16-byte alignment, strides multiples of 8", who);
  p.x = (const __bf16*)a->x; p.weight = (const __bf16*)a->weight; p.out = (__bf16*)a->out;
  p.x_ts = a->x_ts; p.x_hs = a->x_hs; p.out_ts = a->out_ts; p.out_hs = a->out_hs;
  p.T = (int)a->T; p.H = (int)a->H;
  return PITH_OK;
}

// Token blocks for a grid of `columns` workgroups each: as many as give every compute unit a workgroup (which reads its weights anew), of whole tiles.
int tokens_per_block(int T, int tile, int columns) {
  const int tiles = (T + tile - 1) / tile, want = std::max(1, compute_units_or_default() / columns);
  return tile * ((tiles + want - 1) / want);
}

unsigned grid_of(int64_t work, int64_t each) { return (unsigned)((work + each - 1) / each); }

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int pith_latent_absorb_query(const pith_latent_absorb_args* a, pith_stream_t stream) {
  const char* who = "pith_latent_absorb_query";
  AbsorbParams p = {};
  if (const int rc = check_absorb(a, who, kNope + kRope, kLatent, p)) return rc;
  if (a->P < 1) return fail(PITH_ERR_BAD_SHAPE, "%s: tables of %lld positions", who, (long long)a->P);
  if (a->T == 0) return PITH_OK;
  if (!a->q_pe || !a->cos || !a->sin || !a->position_ids) return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if ((a->T > 1 && a->q_pe_ts < kRope) || (a->H > 1 && a->q_pe_hs < kRope)) return fail(PITH_ERR_BAD_SHAPE, "%s: a stride of q_pe is shorter than its features", who);
  if (!aligned16(a->q_pe) || (a->q_pe_ts | a->q_pe_hs) % 8 || (uintptr_t)a->position_ids % 8 || (uintptr_t)a->cos % 2 || (uintptr_t)a->sin % 2)
    return fail(PITH_ERR_MISALIGNED, "%s: q_pe needs 16-byte alignment and strides of multiples of 8, position_ids 8-byte alignment", who);
  p.q_pe = (__bf16*)a->q_pe; p.q_pe_ts = a->q_pe_ts; p.q_pe_hs = a->q_pe_hs;
  p.cos = (const __bf16*)a->cos; p.sin = (const __bf16*)a->sin; p.pos = a->position_ids; p.P = a->P;
  const int64_t pairs = (int64_t)p.T * p.H * (kRope / 2);
  // More than four tiles of 32 tokens and a head a compute unit: whole heads by one workgroup a unit, and the rotation in a launch of its own (beside
  // 136 KB of LDS it would have a unit to a workgroup). Fewer: a quarter of a head to a workgroup of two waves, all in one launch. In us, 8 waves + rotation
  // / 2 waves: 16 heads, 32 tokens 5.5 + 2.9 / 3.7, 512 tokens 8.3 + 4.0 / 9.7, 2048 tokens 14.4 + 4.3 / 16.5; 128 heads, 1 token 8.0 + 3.9 / 6.0, 256 tokens
  // 15.9 + 4.5 / 20.3, 512 tokens 22.3 + 7.2 / 35.7, 2048 tokens 82 + 24 / 138.
  const int tiles = (p.T + 31) / 32;
  p.tokens_per_block = tokens_per_block(p.T, 32, p.H);
  const unsigned blocks = grid_of(p.T, p.tokens_per_block), eights = grid_of((int64_t)p.H * blocks, 8);
  begin_launch();
  if ((int64_t)tiles * p.H > 4 * compute_units_or_default()) {
    absorb_query_kernel<8><<<8 * eights, 512, 0, (hipStream_t)stream>>>(p, 8 * eights, (int)blocks);
    absorb_rotate_kernel<<<grid_of(pairs, kPairs * kRotateThreads), kRotateThreads, 0, (hipStream_t)stream>>>(p);
  } else {
    absorb_query_kernel<2><<<32 * eights + grid_of(pairs, kPairs * 128), 128, 0, (hipStream_t)stream>>>(p, 32 * eights, (int)blocks);
  }
  return check_launch(who);
}

extern "C" int pith_latent_absorb_value(const pith_latent_absorb_args* a, pith_stream_t stream) {
  const char* who = "pith_latent_absorb_value";
  AbsorbParams p = {};
  if (const int rc = check_absorb(a, who, kLatent, kValue, p)) return rc;
  if (a->T == 0) return PITH_OK;
  // Tiles of sixteen tokens and a head for four a compute unit: all 128 features by one workgroup a unit, whose ring keeps 128 KB in flight. Fewer: two
  // workgroups of 64 features each, for more of them at a time. In us, 8 / 4 waves: 16 heads, 1 token 4.2 / 3.4, 128 tokens 4.8 / 3.9, 512 tokens 7.7 / 8.1;
  // 128 heads, 1 token 6.2 / 5.6, 128 tokens 11.4 / 11.8, 512 tokens 25.3 / 26.8, 2048 tokens 72 / 89.
  const int tiles = (p.T + 15) / 16, units = compute_units_or_default();
  p.tokens_per_block = tokens_per_block(p.T, 16, p.H);
  const unsigned blocks = grid_of(p.T, p.tokens_per_block);
  begin_launch();
  if ((int64_t)tiles * p.H >= 4 * units) absorb_value_kernel<8><<<dim3(1, (unsigned)p.H, blocks), 512, 0, (hipStream_t)stream>>>(p);
  else absorb_value_kernel<4><<<dim3(2, (unsigned)p.H, blocks), 256, 0, (hipStream_t)stream>>>(p);
  return check_launch(who);
}
