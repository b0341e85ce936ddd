// Attention of new tokens to the rows of a latent cache (see latent_attn.h for the work list), 16 query rows to a workgroup.
//
//   S = kappa (Q_latent C^T + Q_pe P^T),  O = softmax(S) C
//
// The 32 rows of a tile come in once (36 KB as bf16, 20 KB as e4m3) and are used twice, as keys and as values, by 16 heads of one token: 30
// (54) flop a byte, far below what the matrix cores need, so the kernel is a stream of cache rows with everything else behind it. Rows are moved
// global -> LDS by direct loads, one row an instruction (bf16), into a ring of tiles; page numbers are scalar loads, two a tile.
// Four wavefronts share a tile twice over:
//   scores  wave w: keys 16 (w & 1) .. of the tile, half w >> 1 of the 576 features. A operand = keys, B operand = query rows (in registers for the
//           whole walk), so a lane owns one query row. The two halves meet in LDS (4 KB), where every wave reads the sums of all 32 keys in the
//           order in which the second product contracts them,
//   softmax by every wave for itself (8 scores a lane: cheaper than another exchange and barrier),
//   result  wave w: features 128 w .. of all 16 rows, values read transposed from the same tile.
// Two barriers a tile.
#include "latent_attn.h"

namespace pith {
namespace {

constexpr int kThreads = 256;
constexpr int kM = 16;  // query rows of a workgroup

template <bool FP8>
struct Tile {
  static constexpr int kLatentRow = FP8 ? kLatent : 2 * kLatent;       // bytes
  static constexpr int kPe = kLatentKeys * kLatentRow;                 // offsets in a tile
  static constexpr int kScale = kPe + kLatentKeys * 2 * kRope;         // [4 waves][64] fp32, wave-private copies (the second 32 repeat)
  static constexpr int kBytes = kScale + (FP8 ? 1024 : 0);
  static constexpr int kLoads = FP8 ? 6 : 9;                           // direct loads of a wave
};

template <bool FP8>
constexpr int kStages = FP8 ? 3 : 2;
constexpr int kScoreRow = 36;  // floats of a row of the score exchange: 32 keys and 4 that spread the rows over the banks
constexpr int kScoreBytes = 2 * kM * kScoreRow * 4;

template <bool FP8>
constexpr int kLdsBytes = kStages<FP8> * Tile<FP8>::kBytes + kScoreBytes;

// Piece (16 bytes) swizzle of latent row r: sixteen consecutive rows read at one piece hit different banks, and rows r .. r+3 different 64-byte
// groups (attn_tiles.h). Rows are whole multiples of 256 bytes, so it acts on the low four bits of the piece.
__device__ __forceinline__ int swz(int row) { return tile_swizzle(row); }

// Page entry of tile row 0 or 16 of the tile whose first key is key0; entries behind the sequence's last row count as that row's.
__device__ __forceinline__ int page_of(const LatentAttnParams& p, const int32_t* table, int key, int len) {
  const int k = min(key, max(len - 1, 0));
  return safe_page(table[k >> p.cache.page_shift], p.cache.pages);
}

// Issues the wave's direct loads of one tile. Wave w moves tile rows 4w..4w+3 and 16+4w..; rows behind the last one are read as that one.
template <bool FP8>
__device__ __forceinline__ void issue_tile(const LatentAttnParams& p, int page_lo, int page_hi, int key0, int len, char* slot, int wave, int lane) {
  const int in_mask = (1 << p.cache.page_shift) - 1;
  const int last = max(len - 1, 0);
  using T = Tile<FP8>;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int page = half ? page_hi : page_lo;
    const int first = min(key0 + 16 * half, last) & ~15;  // of the 16 rows around it, which share a page
    const char* const base = p.cache.latent + page * p.cache.latent_ps + (int64_t)(first & in_mask) * T::kLatentRow;
    const int left = last - first;  // rows behind `first` that exist
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // two rows an instruction
        const int r = 4 * wave + 2 * i + (lane >> 5);
        const int piece = (lane & 31) ^ swz(16 * half + r);
        load_lds16(base, min(r, left) * T::kLatentRow + 16 * piece, slot + (16 * half + 4 * wave + 2 * i) * T::kLatentRow);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * wave + i;
        load_lds16(base + min(r, left) * T::kLatentRow, 16 * (lane ^ swz(16 * half + r)), slot + (16 * half + r) * T::kLatentRow);
      }
    }
  }
  // rotary parts: LDS row r (256 bytes) holds tile rows r and r + 16 in pieces 0-7 and 8-15
  const int r = 4 * wave + (lane >> 4);
  const int piece = (lane & 15) ^ swz(r);
  const bool hi = piece >= 8;
  {
    const int first_lo = min(key0, last) & ~15, first_hi = min(key0 + 16, last) & ~15;
    const int first = hi ? first_hi : first_lo;
    const int64_t page = hi ? page_hi : page_lo;
    const char* src = reinterpret_cast<const char*>(p.cache.k_pe + page * p.cache.k_pe_ps + (int64_t)((first & in_mask) + min(r, last - first)) * kRope) + 16 * (piece & 7);
    load_lds16_at(src, slot + T::kPe + wave * 1024);
  }
  if constexpr (FP8) {
    const int k = min(key0 + (lane & 31), last);
    const int64_t page = (lane & 16) ? page_hi : page_lo;
    load_lds4(p.cache.scale + page * p.cache.scale_ps + (k & in_mask), slot + T::kScale + wave * 256);
  }
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// max / sum over the four lanes c, c + 16, c + 32, c + 48 that share a query row
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <int LATER>
__device__ __forceinline__ void wait_loads() {
  static_assert(LATER < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (LATER & 15) | ((LATER >> 4) << 14));
  asm volatile("" ::: "memory");
}

// Which feature of the wave's 128 result v of product n is in a lane of group g. Transposed reads take their columns in groups of four (bf16) or
// eight (e4m3) from wherever a lane points; as bf16 the groups of two products are dealt so that a lane's results of both are eight consecutive ones.
template <bool FP8>
__device__ __forceinline__ int feature_of(int n, int g) {
  return FP8 ? 16 * n + 4 * g : 32 * (n >> 1) + 8 * g + 4 * (n & 1);
}

// A operand of product n: features of the wave's 128 (from f0 on) as rows, keys 8 g + e as contraction.
template <bool FP8>
__device__ __forceinline__ bf16x8 value_fragment(const char* tile, int f0, int n, int c, int g) {
  if constexpr (FP8) {
    typedef __attribute__((ext_vector_type(2))) int i32x2;
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    const int r = 8 * g + (c >> 1), feature = f0 + 16 * n + 8 * (c & 1);
    const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(tile + r * kLatent + (((feature >> 4) ^ swz(r)) << 4) + (feature & 15)));
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bf16x2 two = (e & 1) ? fp8x2_to_bf16<true>(raw[e >> 1]) : fp8x2_to_bf16<false>(raw[e >> 1]);
      v[2 * e] = two[0];
      v[2 * e + 1] = two[1];
    }
    return v;
  } else {
    const int r = 8 * g + (c >> 2), feature = f0 + feature_of<false>(n, c & 3);
    return lds_read_transposed_at(tile + r * 2 * kLatent + (((feature >> 3) ^ swz(r)) << 4) + ((feature & 7) << 1),
                                  tile + (r + 4) * 2 * kLatent + (((feature >> 3) ^ swz(r + 4)) << 4) + ((feature & 7) << 1));
  }
}

// Infinities and NaN -> 0. For tiles that some rows see in part only: a row's weight of a key it does not see is 0, and must stay so against whatever
// the key holds. A row that sees such a key has a score of the same kind.
__device__ __forceinline__ bf16x8 finite(bf16x8 v) {
  u32x4 x = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u;
    if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0xffffu;
  }
  return __builtin_bit_cast(bf16x8, x);
}

template <bool FP8, bool TREE>
__global__ __launch_bounds__(kThreads, 2) void latent_attn_kernel(LatentAttnParams p) {
  using T = Tile<FP8>;
  constexpr int kRing = kStages<FP8>;
  __shared__ __attribute__((aligned(1024))) char lds[kLdsBytes<FP8>];
  float* const scores = reinterpret_cast<float*>(lds + kRing * T::kBytes);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;

  // ---- the range of this workgroup: sums over the sequences, by every wave for itself
  int total = 0, blocks_total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    int w = 0, k = 0;
    if (b0 + lane < p.B) {
      const SeqWork s = seq_work(p, b0 + lane, kM);
      w = s.blocks * s.tiles;
      k = s.blocks;
    }
    total += __builtin_amdgcn_readlane(wave_scan(w, lane), 63);
    blocks_total += __builtin_amdgcn_readlane(wave_scan(k, lane), 63);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.items = min(blocks_total, p.max_items);
  const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, p.min_tiles);
  const int begin = blockIdx.x * per, end = min(begin + per, total);  // (the host has bounded total + gridDim * min_tiles)
  if (begin >= end) return;
  int b = 0, before = 0, item = 0;  // sequence of the first tile, tiles and row blocks in front of it
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    int w = 0, k = 0;
    if (b0 + lane < p.B) {
      const SeqWork s = seq_work(p, b0 + lane, kM);
      w = s.blocks * s.tiles;
      k = s.blocks;
    }
    const int sw = wave_scan(w, lane), sk = wave_scan(k, lane);
    const uint64_t beyond = __ballot(before + sw > begin);
    if (beyond != 0) {
      const int i = __builtin_ctzll(beyond);
      b = b0 + i;
      before += __builtin_amdgcn_readlane(sw - w, i);
      item += __builtin_amdgcn_readlane(sk - k, i);
      break;
    }
    before += __builtin_amdgcn_readlane(sw, 63);
    item += __builtin_amdgcn_readlane(sk, 63);
  }
  b = __builtin_amdgcn_readfirstlane(b);
  SeqWork s = seq_work(p, b, kM);
  int block = (begin - before) / s.tiles;
  int tile = begin - before - block * s.tiles;
  item += block;

  for (int at = begin; at < end;) {
    const int n_tiles = min(s.tiles - tile, end - at);
    const int row0 = block * kM, rows = min(s.n * p.H - row0, kM);
    const int row = row0 + min(c, rows - 1);
    const int tok = row / p.H, head = row - tok * p.H;
    const int32_t* const table = p.table + b * p.table_rs;
    const int ctx = s.len - s.n;  // rows in front of the new ones (below zero only where the lengths contradict each other)

    // ---- queries: pieces 4 st + g of the row, this wave's half of the steps. e4m3 keys are read 16 features at a time: latent steps 2 i, 2 i + 1
    // then contract features 64 i + 16 g + {0..7, 8..15}.
    const int half = wave >> 1, kg = wave & 1;
    constexpr int kSteps = FP8 ? 10 : 9;  // of the longer half (e4m3: 8 and 8 latent, 2 rotary)
    bf16x8 q[kSteps];
    {
      const __bf16* ql = p.q_latent + (int64_t)(s.tok0 + tok) * p.q_ts + head * p.q_hs;
      const __bf16* qp = p.q_pe + (int64_t)(s.tok0 + tok) * p.q_pe_ts + head * p.q_pe_hs;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if constexpr (FP8) {
          if (i < 8) q[i] = *reinterpret_cast<const bf16x8*>(ql + 256 * half + 64 * (i >> 1) + 16 * g + 8 * (i & 1));
          else q[i] = *reinterpret_cast<const bf16x8*>(qp + 32 * (i - 8) + 8 * g);
        } else {
          const int st = 9 * half + i;
          q[i] = *reinterpret_cast<const bf16x8*>(st < 16 ? ql + 32 * st + 8 * g : qp + 32 * (st - 16) + 8 * g);
        }
      }
    }
    uint64_t word = 0;
    if constexpr (TREE) word = (uint64_t)p.tree[s.tok0 + tok];

    f32x4 acc[8] = {};
    float m = -INFINITY, l = 0.f;

    __syncthreads();  // the ring's slots are free: every wave is through with the row block before
    const int key_first = tile * kLatentKeys;
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i)
      if (i < n_tiles) {
        const int key0 = key_first + i * kLatentKeys;
        issue_tile<FP8>(p, page_of(p, table, key0, s.len), page_of(p, table, key0 + 16, s.len), key0, s.len, lds + i * T::kBytes, wave, lane);
      }
    int next_lo = page_of(p, table, key_first + (kRing - 1) * kLatentKeys, s.len), next_hi = page_of(p, table, key_first + (kRing - 1) * kLatentKeys + 16, s.len);
    int slot = 0;
    for (int i = 0; i < n_tiles; ++i) {
      const int key0 = key_first + i * kLatentKeys;
      if (kRing == 2 || i + 1 >= n_tiles) wait_loads<0>();
      else wait_loads<(kRing - 2) * T::kLoads>();
      __syncthreads();
      if (i + kRing - 1 < n_tiles) {
        const int key = key0 + (kRing - 1) * kLatentKeys;
        int into = slot + kRing - 1;
        into = into >= kRing ? into - kRing : into;
        issue_tile<FP8>(p, next_lo, next_hi, key, s.len, lds + into * T::kBytes, wave, lane);
        next_lo = page_of(p, table, key + kLatentKeys, s.len);
        next_hi = page_of(p, table, key + kLatentKeys + 16, s.len);
      }
      const char* const kt = lds + slot * T::kBytes;
      slot = slot + 1 == kRing ? 0 : slot + 1;

      // ---- scores of 16 keys, half of the features
      {
        const int kr = 16 * kg + c;  // the key this lane brings
        const char* const krow = kt + kr * T::kLatentRow;
        const char* const prow = kt + T::kPe + c * 256;
        f32x4 a0 = {}, a1 = {};
        if constexpr (FP8) {
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            const u32x4 raw = *reinterpret_cast<const u32x4*>(krow + (((16 * half + 4 * i2 + g) ^ swz(kr)) << 4));
            bf16x8 k0, k1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bf16x2 x = (e & 1) ? fp8x2_to_bf16<true>(raw[e >> 1]) : fp8x2_to_bf16<false>(raw[e >> 1]);
              const bf16x2 y = (e & 1) ? fp8x2_to_bf16<true>(raw[2 + (e >> 1)]) : fp8x2_to_bf16<false>(raw[2 + (e >> 1)]);
              k0[2 * e] = x[0]; k0[2 * e + 1] = x[1];
              k1[2 * e] = y[0]; k1[2 * e + 1] = y[1];
            }
            a0 = mfma16(k0, q[2 * i2], a0);
            a1 = mfma16(k1, q[2 * i2 + 1], a1);
          }
          const f32x4 sc = *reinterpret_cast<const f32x4*>(kt + T::kScale + wave * 256 + (16 * kg + 4 * g) * 4);
          a0 = (a0 + a1) * sc;
          if (half) {  // wave-uniform
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
              const bf16x8 k = *reinterpret_cast<const bf16x8*>(prow + (((8 * kg + 4 * i2 + g) ^ swz(c)) << 4));
              a0 = mfma16(k, q[8 + i2], a0);
            }
          }
        } else {
#pragma unroll
          for (int i2 = 0; i2 < 9; ++i2) {
            const int st = 9 * half + i2;
            const char* const src = st < 16 ? krow + (((4 * st + g) ^ swz(kr)) << 4) : prow + (((8 * kg + 4 * (st - 16) + g) ^ swz(c)) << 4);
            const bf16x8 k = *reinterpret_cast<const bf16x8*>(src);
            if (i2 & 1) a1 = mfma16(k, q[i2], a1);
            else a0 = mfma16(k, q[i2], a0);
          }
          a0 += a1;
        }
        *reinterpret_cast<f32x4*>(scores + (half * kM + c) * kScoreRow + 16 * kg + 4 * g) = a0;
      }
      __syncthreads();

      // ---- softmax of the row's keys 8 g .. 8 g + 7
      float x[8];
      {
        const f32x4* const r0 = reinterpret_cast<const f32x4*>(scores + c * kScoreRow + 8 * g);
        const f32x4* const r1 = reinterpret_cast<const f32x4*>(scores + (kM + c) * kScoreRow + 8 * g);
        const f32x4 lo = r0[0] + r1[0], hi = r0[1] + r1[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = lo[e] * p.kappa, x[4 + e] = hi[e] * p.kappa;
      }
      const bool partial = key0 + kLatentKeys > ctx + (TREE ? 0 : 1);  // some row may not see all of the tile
      if (partial) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + 8 * g + e;
          bool seen = key < s.len;
          if constexpr (TREE) seen = seen && (key < ctx || (key - ctx < 64 && ((word >> ((key - ctx) & 63)) & 1)));
          else seen = seen && key <= ctx + tok;
          x[e] = seen ? x[e] : -INFINITY;
        }
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
      const float m_new = fmaxf(m, quad_max(top));
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      if (__any(m_new > m)) {
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        l *= alpha;
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[n] *= alpha;
        m = m_new;
      }
      float pr[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pr[e] = __builtin_amdgcn_exp2f(x[e] - ref);
        l += pr[e];
      }
      if constexpr (FP8) {
        const f32x4* const sc = reinterpret_cast<const f32x4*>(kt + T::kScale + wave * 256 + 8 * g * 4);
        const f32x4 lo = sc[0], hi = sc[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] *= lo[e], pr[4 + e] *= hi[e];
      }
      const bf16x8 pb = to_bf16x8(pr[0], pr[1], pr[2], pr[3], pr[4], pr[5], pr[6], pr[7]);

      // ---- features 128 wave .. + 127, 16 a product
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        bf16x8 v = value_fragment<FP8>(kt, 128 * wave, n, c, g);
        if (partial && s.n > 1) v = finite(v);  // (wave-uniform)
        acc[n] = mfma16(v, pb, acc[n]);
      }
    }

    // ---- the row block's result, or this part of it
    l = quad_sum(l);
    const bool whole = n_tiles == s.tiles;
    if (whole) {
      if (c < rows) {
        const float inv = 1.f / l;
        __bf16* const dst = p.o + (int64_t)(s.tok0 + tok) * p.o_ts + head * p.o_hs + 128 * wave;
#pragma unroll
        for (int n = 0; n < 8; n += 2) {
          const f32x4 a = l == 0.f ? f32x4{} : acc[n] * inv, d = l == 0.f ? f32x4{} : acc[n + 1] * inv;
          const u32x2 lo = {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3])}, hi = {pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3])};
          if constexpr (FP8) {
            *reinterpret_cast<u32x2*>(dst + feature_of<true>(n, g)) = lo;
            *reinterpret_cast<u32x2*>(dst + feature_of<true>(n + 1, g)) = hi;
          } else {
            *reinterpret_cast<u32x4*>(dst + feature_of<false>(n, g)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
          }
        }
        if (wave == 0 && g == 0) p.lse[head * p.lse_hs + s.tok0 + tok] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
      }
    } else {
      const int64_t part = 2 * blockIdx.x + (at == begin ? 0 : 1);
      float* const dst = p.parts + (part * kM + c) * kLatent + 128 * wave;
#pragma unroll
      for (int n = 0; n < 8; ++n) *reinterpret_cast<f32x4*>(dst + feature_of<FP8>(n, g)) = acc[n];
      if (wave == 0 && g == 0) p.stats[part * kM + c] = make_float2(m, l);
    }
    if (tile + n_tiles == s.tiles && threadIdx.x == 0 && item < p.max_items) {  // who ends a row block says where its parts lie
      const int first_tile = at + n_tiles - s.tiles;  // of the whole work list
      const int g0 = whole ? 0 : first_tile / per;
      p.joins[item] = make_int4(s.tok0 * p.H + row0, rows, whole ? 0 : 2 * g0 + (first_tile == g0 * per ? 0 : 1), whole ? 0 : 2 * (int)blockIdx.x);
    }

    at += n_tiles;
    tile = 0;
    ++item;
    if (++block >= s.blocks && at < end) {
      block = 0;
      do s = seq_work(p, ++b, kM); while (s.blocks == 0);
    }
  }
}

// Joins the parts of a row block: o = sum_i w_i O_i / sum_i w_i l_i, w_i = 2^(m_i - max m). blockIdx.x: row block, blockIdx.y: which of gridDim.y
// shares of its M x 512 results (a share is consecutive pieces of four features); threads beyond a share's pieces take every other part of them.
__global__ __launch_bounds__(kThreads) void latent_join_kernel(LatentAttnParams p) {
  __shared__ __attribute__((aligned(16))) float sum_o[kThreads][4];
  __shared__ float sum_l[kThreads], sum_m[kThreads];
  if ((int)blockIdx.x >= *p.items) return;
  const int4 join = p.joins[blockIdx.x];
  if (join.z == join.w) return;
  const int pieces = kM * kLatent / 4 / gridDim.y;  // of this share: a power of two
  const int lanes = min(pieces, kThreads), groups = kThreads / lanes;
  const int mine = threadIdx.x % lanes, group = threadIdx.x / lanes;
  const int n_parts = join.w / 2 - join.z / 2 + 1;  // slots z, then the even ones up to w
  for (int piece0 = 0; piece0 < pieces; piece0 += lanes) {
    const int piece = blockIdx.y * pieces + piece0 + mine;
    const int row = piece / (kLatent / 4), feature = 4 * (piece % (kLatent / 4));
    float m = -INFINITY, l = 0.f;
    f32x4 o = {};
    for (int i = group; i < n_parts; i += groups) {
      const int64_t slot = i == 0 ? join.z : 2 * (join.z / 2 + i);
      const float2 st = p.stats[slot * kM + row];
      const f32x4 x = *reinterpret_cast<const f32x4*>(p.parts + (slot * kM + row) * kLatent + feature);
      const float m_new = fmaxf(m, st.x);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float old = __builtin_amdgcn_exp2f(m - ref), add = __builtin_amdgcn_exp2f(st.x - ref);
      o = o * old + x * add;
      l = l * old + st.y * add;
      m = m_new;
    }
    if (groups > 1) {
      *reinterpret_cast<f32x4*>(sum_o[threadIdx.x]) = o;
      sum_l[threadIdx.x] = l;
      sum_m[threadIdx.x] = m;
      __syncthreads();
      if (group == 0) {
        float top = m;
        for (int k = 1; k < groups; ++k) top = fmaxf(top, sum_m[k * lanes + mine]);
        const float ref = top == -INFINITY ? 0.f : top;
        const float w0 = __builtin_amdgcn_exp2f(m - ref);
        o *= w0;
        l *= w0;
        for (int k = 1; k < groups; ++k) {
          const float w = __builtin_amdgcn_exp2f(sum_m[k * lanes + mine] - ref);
          o += *reinterpret_cast<const f32x4*>(sum_o[k * lanes + mine]) * w;
          l += sum_l[k * lanes + mine] * w;
        }
        m = top;
      }
    }
    if (group == 0 && row < join.y) {
      const int r = join.x + row, tok = r / p.H, head = r - tok * p.H;
      o = l == 0.f ? f32x4{} : o * (1.f / l);
      const u32x2 out = {pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
      *reinterpret_cast<u32x2*>(p.o + (int64_t)tok * p.o_ts + head * p.o_hs + feature) = out;
      if (feature == 0) p.lse[head * p.lse_hs + tok] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
    }
  }
}

constexpr int kMinTiles = 2;

struct LatentPlan {
  int groups;      // workgroups of the attention kernel
  int max_items;   // row blocks at most
  int join_shares;
  int64_t joins_at, stats_at, parts_at, bytes;  // workspace
};

LatentPlan plan_of(const pith_latent_attn_args* a) {
  LatentPlan pl = {};
  const int64_t rows = a->T * a->H;
  const int64_t items = (rows + kM - 1) / kM + (a->B < a->T ? a->B : a->T);
  pl.max_items = (int)items;
  pl.groups = 2 * compute_units_or_default();
  int shares = 1;
  while (shares < 64 && shares * items < 512) shares *= 2;
  pl.join_shares = shares;
  const auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  pl.joins_at = 256;
  pl.stats_at = pl.joins_at + up(items * (int64_t)sizeof(int4));
  pl.parts_at = pl.stats_at + up((int64_t)2 * pl.groups * kM * sizeof(float2));
  pl.bytes = pl.parts_at + (int64_t)2 * pl.groups * kM * kLatent * 4;
  return pl;
}

int check_attn(const pith_latent_attn_args* a, const char* who) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (a->T < 0 || a->B < 0 || a->H < 1 || a->T > 1 << 20 || a->B > 1 << 20 || a->H > 1024 || a->table_width < 0)
    return fail(PITH_ERR_BAD_SHAPE, "%s: T = %lld, B = %lld (at most 2^20), H = %lld (at most 1024), table_width = %lld", who, (long long)a->T, (long long)a->B, (long long)a->H, (long long)a->table_width);
  if (const int rc = check_cache(a->cache, who)) return rc;
  // counted in 32 bits on the device: rows of a sequence, and the tiles of the whole work list
  const int64_t most = a->table_width > 0 && a->table_width > 0x7fffffff / a->cache.page_size ? -1 : a->table_width * a->cache.page_size;
  if (most < 0 || most > 0x7fffffff - 4096) return fail(PITH_ERR_UNSUPPORTED, "%s: page tables of 2^31 rows or more", who);
  const int64_t items = (a->T * a->H + kM - 1) / kM + a->B;
  if (items * (most / kLatentKeys + 1) > 0x7fffffff - 65536) return fail(PITH_ERR_UNSUPPORTED, "%s: too many row blocks for page tables of that width: call it with fewer tokens at a time", who);
  return PITH_OK;
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int64_t pith_latent_attn_workspace_bytes(const pith_latent_attn_args* a) {
  if (check_attn(a, "pith_latent_attn_workspace_bytes") != PITH_OK || a->T == 0 || a->B == 0) return 0;
  return plan_of(a).bytes;
}

extern "C" int pith_latent_attn(const pith_latent_attn_args* a, pith_stream_t stream) {
  const char* who = "pith_latent_attn";
  if (const int rc = check_attn(a, who)) return rc;
  if (a->T == 0 || a->B == 0) return PITH_OK;
  if (!a->q_latent || !a->q_pe || !a->lengths || !a->cu_q || !a->o || !a->lse || !a->workspace || (!a->page_table && a->table_width > 0))
    return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if (a->table_width == 0) return fail(PITH_ERR_BAD_SHAPE, "%s: an empty page table holds no rows", who);
  if ((a->B > 1 && a->table_rs < a->table_width) || (a->T > 1 && (a->q_ts < kLatent || a->q_pe_ts < kRope || a->o_ts < kLatent)) ||
      (a->H > 1 && (a->q_hs < kLatent || a->q_pe_hs < kRope || a->o_hs < kLatent || a->lse_hs < a->T)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a stride is shorter than what it steps over", who);
  if (!aligned16(a->q_latent) || !aligned16(a->q_pe) || !aligned16(a->o) || (a->q_ts | a->q_hs | a->q_pe_ts | a->q_pe_hs | a->o_ts | a->o_hs) % 8 || (uintptr_t)a->workspace % 256 ||
      (uintptr_t)a->page_table % 4 || (uintptr_t)a->lengths % 4 || (uintptr_t)a->cu_q % 4 || (uintptr_t)a->lse % 4 || (uintptr_t)a->tree_mask % 8)
    return fail(PITH_ERR_MISALIGNED, "%s: queries and results need 16-byte alignment and strides of multiples of 8, the workspace 256-byte alignment", who);
  const LatentPlan pl = plan_of(a);
  if (a->workspace_bytes < pl.bytes) return fail(PITH_ERR_BAD_SHAPE, "%s: the workspace has %lld bytes, %lld are needed", who, (long long)a->workspace_bytes, (long long)pl.bytes);
  LatentAttnParams p = {};
  p.q_latent = (const __bf16*)a->q_latent; p.q_pe = (const __bf16*)a->q_pe;
  p.cache = to_device(a->cache);
  p.table = a->page_table; p.lengths = a->lengths; p.cu_q = a->cu_q; p.tree = a->tree_mask;
  p.o = (__bf16*)a->o; p.lse = a->lse;
  p.table_rs = a->B > 1 ? a->table_rs : 0;
  p.q_ts = a->q_ts; p.q_hs = a->q_hs; p.q_pe_ts = a->q_pe_ts; p.q_pe_hs = a->q_pe_hs; p.o_ts = a->o_ts; p.o_hs = a->o_hs; p.lse_hs = a->lse_hs;
  p.T = (int)a->T; p.B = (int)a->B; p.H = (int)a->H; p.table_width = (int)a->table_width;
  p.max_len = (int)(a->table_width * a->cache.page_size);
  p.kappa = a->scale * 1.4426950408889634f;
  char* const ws = (char*)a->workspace;
  p.items = (int*)ws;
  p.joins = (int4*)(ws + pl.joins_at);
  p.stats = (float2*)(ws + pl.stats_at);
  p.parts = (float*)(ws + pl.parts_at);
  p.max_items = pl.max_items;
  p.min_tiles = kMinTiles;
  const bool fp8 = a->cache.dtype == PITH_FP8_E4M3, tree = a->tree_mask != nullptr;
  hipStream_t s = (hipStream_t)stream;
  begin_launch();
  if (fp8 && tree) latent_attn_kernel<true, true><<<pl.groups, kThreads, 0, s>>>(p);
  else if (fp8) latent_attn_kernel<true, false><<<pl.groups, kThreads, 0, s>>>(p);
  else if (tree) latent_attn_kernel<false, true><<<pl.groups, kThreads, 0, s>>>(p);
  else latent_attn_kernel<false, false><<<pl.groups, kThreads, 0, s>>>(p);
  latent_join_kernel<<<dim3(pl.max_items, pl.join_shares), kThreads, 0, s>>>(p);
  return check_launch(who);
}
