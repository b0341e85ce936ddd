// The products around the absorbed attention: q_nope W_uk into the latent space (with the rotation of q_pe), and W_uv o_latent out of it.
//
// Per head a [T x 128] x [128 x 512] product either way. With few tokens (a decoding step) it is the 4 MB of weights of 16 heads that have to come in,
// with many the queries and results, 1.5 KB a token and head, against 131 kflop: memory in both cases. So a wave takes a share of the output
// features, holds its part of the head's weights in registers as MFMA A operands (each weight is read once per workgroup), and walks the tokens,
// 16 at a time as the B operand (16x16x32: lane = token lane % 16, contraction 8 (lane / 16) + e). The result tile then has the token as its column
// and consecutive features in a lane's registers, so rows leave in 16-byte pieces straight from there.
#include "attn_tiles.h"
#include "latent_common.h"

namespace pith {
namespace {

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

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

constexpr int kQueryThreads = 256;

// q_latent features [128 x, 128 x + 128) of head y, tokens of block z; x = 4: q_pe. W_uk's rows are the contraction (d), so its fragments come
// transposed out of LDS (32 KB, one slice of the head). Wave w owns features 32 w ..: two tiles whose rows are dealt so that a lane's two times
// four results are eight consecutive features (tile n, row 4 g + v: feature 8 g + 4 n + v).
__global__ __launch_bounds__(kQueryThreads) void absorb_query_kernel(AbsorbParams p) {
  __shared__ __attribute__((aligned(16))) char tile[128 * kRowBytes128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y;
  const int t0 = blockIdx.z * p.tokens_per_block, t1 = min(t0 + p.tokens_per_block, p.T);
  if (blockIdx.x == kLatent / 128) {
    for (int i = threadIdx.x; i < (t1 - t0) * (kRope / 2); i += kQueryThreads) {
      const int64_t t = t0 + (i >> 5);
      const int j = i & 31;
      const int64_t at = clamped_position(p.pos[t], p.P) * kRope;
      const uint32_t pair = *reinterpret_cast<const uint32_t*>(p.x + t * p.x_ts + h * p.x_hs + kNope + 2 * j);
      float first, second;
      rotate_pair(pair, p.cos + at, p.sin + at, j, first, second);
      __bf16* dst = p.q_pe + t * p.q_pe_ts + h * p.q_pe_hs;
      dst[j] = (__bf16)first;
      dst[kRope / 2 + j] = (__bf16)second;
    }
    return;
  }
  {
    DirectTile128<128, kQueryThreads> loader;
    loader.init(2 * kLatent, wave, lane);
    loader.issue(reinterpret_cast<const char*>(p.weight + (int64_t)h * (kNope + kValue) * kLatent + 128 * blockIdx.x), 128, tile, wave, lane);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
  }
  const int c = lane & 15, g = lane >> 4;
  bf16x8 w[2][4];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      // lane 4 i + k of a 16-lane group brings four features of row i: group k of the tile's 16
      const int feature = 32 * wave + 8 * (c & 3) + 4 * n;
      const int row = 32 * st + 8 * g + (c >> 2);
      const char* lo = tile + swizzled_offset(row, feature >> 3) + ((feature & 7) << 1);
      const char* hi = tile + swizzled_offset(row + 4, feature >> 3) + ((feature & 7) << 1);
      w[n][st] = lds_read_transposed_at(lo, hi);
    }
  for (int t = t0; t < t1; t += 16) {
    const int mine = t + c;
    const __bf16* src = p.x + (int64_t)min(mine, t1 - 1) * p.x_ts + h * p.x_hs + 8 * g;
    bf16x8 q[4];
#pragma unroll
    for (int st = 0; st < 4; ++st) q[st] = *reinterpret_cast<const bf16x8*>(src + 32 * st);
    f32x4 acc[2] = {};
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int n = 0; n < 2; ++n) acc[n] = mfma16(w[n][st], q[st], acc[n]);
    if (mine < t1) {
      const u32x4 out = {pack_bf16x2(acc[0][0], acc[0][1]), pack_bf16x2(acc[0][2], acc[0][3]), pack_bf16x2(acc[1][0], acc[1][1]), pack_bf16x2(acc[1][2], acc[1][3])};
      *reinterpret_cast<u32x4*>(p.out + (int64_t)mine * p.out_ts + h * p.out_hs + 128 * blockIdx.x + 32 * wave + 8 * g) = out;
    }
  }
}

// o features of head y, tokens of block z. W_uv's rows are contiguous along the contraction, like x's, so both operands come straight from memory.
// A wave owns 32 of the 128 features (two tiles dealt as above), 128 registers of weights.
__global__ __launch_bounds__(256) void absorb_value_kernel(AbsorbParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((blockIdx.x * blockDim.x + threadIdx.x) >> 6);
  const int h = blockIdx.y;
  const int t0 = blockIdx.z * p.tokens_per_block, t1 = min(t0 + p.tokens_per_block, p.T);
  const int c = lane & 15, g = lane >> 4;
  bf16x8 w[2][16];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int feature = 32 * wave + 8 * (c >> 2) + 4 * n + (c & 3);
    const __bf16* src = p.weight + ((int64_t)h * (kNope + kValue) + kNope + feature) * kLatent + 8 * g;
#pragma unroll
    for (int st = 0; st < 16; ++st) w[n][st] = *reinterpret_cast<const bf16x8*>(src + 32 * st);
  }
  for (int t = t0; t < t1; t += 16) {
    const int mine = t + c;
    const __bf16* src = p.x + (int64_t)min(mine, t1 - 1) * p.x_ts + h * p.x_hs + 8 * g;
    bf16x8 x[16];
#pragma unroll
    for (int st = 0; st < 16; ++st) x[st] = *reinterpret_cast<const bf16x8*>(src + 32 * st);
    f32x4 acc[2] = {};
#pragma unroll
    for (int st = 0; st < 16; ++st)
#pragma unroll
      for (int n = 0; n < 2; ++n) acc[n] = mfma16(w[n][st], x[st], acc[n]);
    if (mine < t1) {
      const u32x4 out = {pack_bf16x2(acc[0][0], acc[0][1]), pack_bf16x2(acc[0][2], acc[0][3]), pack_bf16x2(acc[1][0], acc[1][1]), pack_bf16x2(acc[1][2], acc[1][3])};
      *reinterpret_cast<u32x4*>(p.out + (int64_t)mine * p.out_ts + h * p.out_hs + 32 * wave + 8 * g) = out;
    }
  }
}

int check_absorb(const pith_latent_absorb_args* a, const char* who, int in_dim, int out_dim, AbsorbParams& p) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (a->T < 0 || a->T > 1 << 20 || a->H < 1 || a->H > 1024) return fail(PITH_ERR_BAD_SHAPE, "%s: T = %lld tokens, H = %lld heads (at most 2^20, 1024)", who, (long long)a->T, (long long)a->H);
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

// Token blocks: as many as give every compute unit two workgroups, of 16 tokens at least (each reads its weights anew).
int tokens_per_block(int T, int blocks_per_token_block) {
  const int tiles = (T + 15) / 16;
  const int want = (2 * compute_units_or_default() + blocks_per_token_block - 1) / blocks_per_token_block;
  const int per = (tiles + want - 1) / want;
  return 16 * (per < 1 ? 1 : per);
}

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
  p.tokens_per_block = tokens_per_block(p.T, 4 * p.H);
  const dim3 grid(kLatent / 128 + 1, (unsigned)p.H, (unsigned)((p.T + p.tokens_per_block - 1) / p.tokens_per_block));
  begin_launch();
  absorb_query_kernel<<<grid, kQueryThreads, 0, (hipStream_t)stream>>>(p);
  return check_launch(who);
}

extern "C" int pith_latent_absorb_value(const pith_latent_absorb_args* a, pith_stream_t stream) {
  const char* who = "pith_latent_absorb_value";
  AbsorbParams p = {};
  if (const int rc = check_absorb(a, who, kLatent, kValue, p)) return rc;
  if (a->T == 0) return PITH_OK;
  p.tokens_per_block = tokens_per_block(p.T, p.H);
  const dim3 grid(1, (unsigned)p.H, (unsigned)((p.T + p.tokens_per_block - 1) / p.tokens_per_block));
  begin_launch();
  absorb_value_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(p);
  return check_launch(who);
}
