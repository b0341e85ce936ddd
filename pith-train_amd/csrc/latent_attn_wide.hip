// Attention of new tokens to the rows of a latent cache, 64 query rows to a workgroup (see latent_attn.h for the work list, latent_attn.hip for the rest):
// sequences that bring more than 16 rows, by their heads or by several tokens.
//
// A tile of 32 keys is 4.5 Mflop for the 64 rows, 1090 cycles of a compute unit's matrix cores, and 36 KB on its way from memory, so every tile that a
// workgroup fetches serves all 64 rows, and one workgroup of eight waves holds a compute unit. Scoring and adding are given to different waves, one of
// each kind to a SIMD, a tile apart: waves 0-3 have the queries (16 keys of the tile against 32 rows: 144 registers), form the scores of tile i + 1 and its
// weights, and pass these on through LDS; waves 4-7 have the results (128 features of all 64 rows: 128 registers), add tile i's values, and ask for the
// tiles, one request behind every four products. One barrier a tile. So a key fragment is read from LDS by two waves and a value fragment by one, either
// kind of wave fills the other's latencies, and its registers are one operand's. (All eight waves doing both, 16 rows and 64 features each, waited for
// one another and read each key fragment four times: 128 heads 81 us against 74, trees of up to 48 drafts 246 against 217.)
// Trees of up to 48 drafts over 16 sequences of up to 16384 rows, 16 heads (147 GF): 162 us a call; in a kernel trace, median (least), 196 (175) and 11.8 for the
// join. 128 heads over 32 sequences of up to 8192 rows (46 GF, 201 MB): 73 us a call, 64.6 (61.1) and 10.3. From e4m3 172 and 67 us a call. A scoring wave is busy
// for 1700 of a tile's 1850 cycles (half in products, half in softmax), an adding one for 1500, so a scoring wave's chain is the nearest bound; sixteen waves of
// half the size, a higher priority for the scoring ones, and 4, 6 or 8 fragments read ahead all took the same time within 1 %, and why is open.
// All 64 rows of a block are multiplied and weighed, and written as a part, whether the sequence brings them or not: two tokens of 16 heads pay for four.
// Weights are formed against a reference of each row that all waves know from earlier tiles; only a score beyond its slack (kSlack) makes them meet, two
// barriers more, to move it.
#include "latent_attn.h"

#include <type_traits>

namespace pith {
namespace {

// kLeast: parts are 128 KB each, written and read again: drafts of four sequences of 1500 e4m3 rows took 19.2 + 6.6 us (kernel + join) with ranges of 2 tiles,
// 18.5 + 4.9 of 4, 20.5 + 4.7 of 8.
constexpr int kThreads = 512, kM = kWideRows, kKeys = 32, kGroups = kM / 16, kStart = 8, kLeast = 4;

// Two buffers of weights [64 rows][32 keys] bf16, pieces of a row swizzled so that neither the reads (16 rows, piece g or g ^ 1: row_swizzle) nor the
// writes conflict; maxima (or sums) [64 rows][2 key groups] fp32; two stamps: the tile whose scores went beyond their slack.
constexpr int kWeights = kM * kKeys * 2, kMaxima = 2 * kWeights, kStamp = kMaxima + kM * 8, kExchangeBytes = kStamp + 16;
__device__ __forceinline__ int weight_at(int row, int piece) {
  const int four = (row >> 2) & 3;
  return row * (kKeys * 2) + ((piece ^ (((four ^ (four >> 1)) & 1) << 1 | four >> 1)) << 4);
}

template <bool FP8, bool TREE>
__global__ __launch_bounds__(kThreads, 2) void latent_attn_wide_kernel(LatentAttnParams p) {
  using T = LatentTile<FP8, kKeys>;
  using Loads = TileLoads<FP8, kKeys>;
  constexpr int kRing = FP8 ? 6 : 4;
  constexpr int J = 2;                // groups of 16 rows that a scoring wave has
  constexpr int Q = kLatent / 32 + 2;  // query fragments, the last two rotary
  __shared__ __attribute__((aligned(1024))) char lds[kRing * T::kBytes + kExchangeBytes];
  static_assert((kRing - 1) * T::kBytes >= LatentTile<false, kM>::kBytes, "the queries are staged in what the first tile leaves of the ring");
  char* const staged = lds + T::kBytes;
  char* const exchange = lds + kRing * T::kBytes;
  int* const stamp = reinterpret_cast<int*>(exchange + kStamp);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Walk<kM, kKeys, kStart, kLeast> walk;
  if (!walk.start(p, threadIdx.x & 63)) return;

  do {
    const SeqWork& s = walk.s;
    const int n_tiles = walk.n_tiles();
    __syncthreads();  // the ring's slots and the exchange are free: every wave is through with the segment before
    if (threadIdx.x < 2) stamp[threadIdx.x] = -1;

    if (wave < 4) {
      stage_queries<kM>(p, walk, staged, wave, lane_here());
      // Scores and weights of keys 16 kg .. of every tile, rows 32 set ..
      const int lane = lane_here(), c = lane & 15, g = lane >> 4;  // (formed in each role: what follows from it takes no register in the other)
      const int kg = wave & 1, set = wave >> 1;
      const int key_row = 16 * kg + c;  // the key this lane brings
      const int key_at = key_row * T::kLatentRow + ((g ^ row_swizzle(key_row)) << 4);
      const int pe_at = T::kPe + pe_row(key_row) * 256 + (((8 * ((key_row >> 2) & 1) + g) ^ pe_swizzle(pe_row(key_row))) << 4);
      bf16x8 q[J][Q];
      wait_loads<0>();
      __syncthreads();  // (1) the queries are there
#pragma unroll
      for (int j = 0; j < J; ++j) read_query<FP8, kM>(staged, 16 * (J * set + j) + c, 0, g, q[j]);
      __syncthreads();  // (2) and have been read

      f32x4 x[J], sc = {};       // scores of a tile, scales of its keys
      float factor = p.kappa;    // what the scores are still to be multiplied by
      float m[J], ref[J], l[J];  // references of the lane's rows, the same to subtract (0 while there is none), and sums over its keys
#pragma unroll
      for (int j = 0; j < J; ++j) m[j] = -INFINITY, ref[j] = l[j] = 0.f;
      const auto tile_scores = [&](const char* kt, f32x4 (&y)[J]) __attribute__((always_inline)) {
        constexpr int kLatentReads = FP8 ? kLatent / 64 : kLatent / 32, kReads = kLatentReads + 2, kAhead = 4;  // fragments read ahead of their products
        const uint32_t first = lds_address(kt) + key_at, pe_first = lds_address(kt) + pe_at;
        const auto read = [&](int n) __attribute__((always_inline)) {
          return n < kLatentReads ? *lds_at<u32x4>((first ^ (64 * (n & 3))) + 256 * (n >> 2)) : *lds_at<u32x4>(pe_first ^ (64 * (n - kLatentReads)));
        };
        if constexpr (FP8) sc = *reinterpret_cast<const f32x4*>(kt + T::kScale + (16 * kg + 4 * g) * 4);
        u32x4 k[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) k[n] = read(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < J; ++j) y[j] = f32x4{};
#pragma unroll
        for (int n = 0; n < kReads; ++n) {
          const u32x4 raw = k[n % kAhead];
          if (FP8 && n < kLatentReads) {  // sixteen features a lane: two products
            const bf16x8 k0 = widen(raw[0], raw[1]), k1 = widen(raw[2], raw[3]);
#pragma unroll
            for (int j = 0; j < J; ++j) y[j] = mfma16(k0, q[j][2 * n], y[j]);
#pragma unroll
            for (int j = 0; j < J; ++j) y[j] = mfma16(k1, q[j][2 * n + 1], y[j]);
          } else {
#pragma unroll
            for (int j = 0; j < J; ++j) {
              if (FP8 && n == kLatentReads) y[j] *= sc;
              y[j] = mfma16(__builtin_bit_cast(bf16x8, raw), q[j][Q - kReads + n], y[j]);
            }
          }
          if (n + kAhead < kReads) k[n % kAhead] = read(n + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // Weights of tile i against the references as they are; what they add to the sums.
      const auto leave_weights = [&](int i, float (&sum)[J], const f32x4& scale) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          f32x4 w;
#pragma unroll
          for (int v = 0; v < 4; ++v) w[v] = __builtin_amdgcn_exp2f(fmaf(x[j][v], factor, -ref[j]));
          sum[j] = (w[0] + w[1]) + (w[2] + w[3]);
          if constexpr (FP8) {
#pragma unroll
            for (int v = 0; v < 4; ++v) w[v] = scaled(w[v], scale[v]);
          }
          *reinterpret_cast<u32x2*>(exchange + (i & 1) * kWeights + weight_at(c, 2 * kg + (g >> 1)) + 16 * (J * set + j) * (kKeys * 2) + 8 * (g & 1)) =
              u32x2{pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])};
        }
      };
      const auto weigh = [&](int i, float (&sum)[J]) __attribute__((always_inline)) {  // scores x of tile i
        const int key0 = (walk.tile + i) * kKeys;
        bool beyond = false;
        factor = p.kappa;
        if (partial_tile<TREE, kKeys>(s, key0) || p.kappa < 0.f) {  // (below zero the largest score is not the largest product)
          factor = 1.f;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            x[j] *= p.kappa;
            if (partial_tile<TREE, kKeys>(s, key0))
              mask_scores<TREE, 4>(p, s, x[j], (walk.block * kM + min(16 * (J * set + j) + c, walk.rows(p) - 1)) / p.H, key0 + 16 * kg + 4 * g);
          }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) beyond |= fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])) * factor > m[j] + kSlack;
        leave_weights(i, sum, sc);
        if (__any(beyond) && lane == 0) stamp[i & 1] = i;
      };

      float sum[J];
      __syncthreads();  // (3) the first tile is there
      tile_scores(lds, x);
      weigh(0, sum);
      int slot = 0;
      for (int i = 0; i < n_tiles; ++i) {
        __syncthreads();  // (4) tile i + 1 is there, and the weights of tile i are
        slot = slot + 1 == kRing ? 0 : slot + 1;
        const int marked = stamp[i & 1];
        const f32x4 scale = sc;
        f32x4 next[J];
        if (i + 1 < n_tiles) tile_scores(lds + slot * T::kBytes, next);
        if (__builtin_amdgcn_readfirstlane(marked) == i) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const float top = quad_max(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3]))) * factor;
            if (g == 0) *reinterpret_cast<float*>(exchange + kMaxima + 8 * (16 * (J * set + j) + c) + 4 * kg) = top;
          }
          __syncthreads();  // (5)
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const f32x2 k = *reinterpret_cast<const f32x2*>(exchange + kMaxima + 8 * (16 * (J * set + j) + c));
            const float m_new = moved(m[j], fmaxf(k[0], k[1]));
            l[j] *= m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[j] - m_new);
            m[j] = m_new;
            ref[j] = m_new == -INFINITY ? 0.f : m_new;
          }
          leave_weights(i, sum, scale);
          __syncthreads();  // (6)
        }
#pragma unroll
        for (int j = 0; j < J; ++j) l[j] += sum[j];
        if (i + 1 < n_tiles) {
#pragma unroll
          for (int j = 0; j < J; ++j) x[j] = next[j];
          weigh(i + 1, sum);
        }
      }
      __syncthreads();  // (7) the last maxima have been read
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float part = quad_sum(l[j]);
        if (g == 0) *reinterpret_cast<float*>(exchange + kMaxima + 8 * (16 * (J * set + j) + c) + 4 * kg) = part;
      }
      __syncthreads();  // (8)
    } else {
      // The tiles' loads, and the results of features 128 w .. of all rows.
      const int lane = lane_here(), c = lane & 15, g = lane >> 4;
      const int w = wave - 4, last = max(s.len - 1, 0);
      const ScalarTable table = (ScalarTable)(uintptr_t)(p.table + walk.b * p.table_rs);
      const int key16 = walk.tile * kKeys + 16 * (w >> 1);  // the sixteen among which this wave's rows of the first tile are
      const auto request = [&](int i) __attribute__((always_inline)) {
        const int key = key16 + i * kKeys;
        Loads(p, page_at(p, table, key, last), key, last, lds + i * T::kBytes, w).issue_all(lane);
      };
      request(0);
      int next_page = page_at(p, table, key16 + (kRing - 1) * kKeys, last);
      f32x4 acc[kGroups][8] = {};
      float m[kGroups];  // references of the lane's row of every group
#pragma unroll
      for (int r = 0; r < kGroups; ++r) m[r] = -INFINITY;
      stage_queries<kM>(p, walk, staged, wave, lane_here());
      wait_loads<0>();
      __syncthreads();  // (1)
      __syncthreads();  // (2)
#pragma unroll 1
      for (int i = 1; i < min(kRing - 1, n_tiles); ++i) request(i);
      if (n_tiles >= kRing - 1) wait_loads<(kRing - 2) * Loads::kLoads>();
      else wait_loads<0>();
      __syncthreads();  // (3)
      const int value_at = value_place<FP8>(w, c, g);
      int slot = 0;
      const auto add = [&](int i, auto more) __attribute__((always_inline)) {  // tile i
        char* const kt = lds + slot * T::kBytes;
        char* const into = lds + (slot == 0 ? kRing - 1 : slot - 1) * T::kBytes;
        slot = slot + 1 == kRing ? 0 : slot + 1;
        const int key = key16 + (i + kRing - 1) * kKeys;
        const Loads loads(p, next_page, key, last, into, w);
        if (more || i + kRing - 2 < n_tiles) wait_loads<(kRing - 3) * Loads::kLoads>();
        else wait_loads<0>();
        __syncthreads();  // (4) nobody reads tile i - 1 any more
        const int marked = stamp[i & 1];
        constexpr int kAhead = 4;  // products whose values are read ahead
        const uint32_t values = lds_address(kt) + value_at;
        bf16x8 weight[kGroups], v[kAhead];  // weights: keys 8 g + e of the lane's row of each group
        const auto read_first = [&]() __attribute__((always_inline)) {
#pragma unroll
          for (int r = 0; r < kGroups; ++r) weight[r] = *reinterpret_cast<const bf16x8*>(exchange + (i & 1) * kWeights + weight_at(c, g) + 16 * r * (kKeys * 2));
#pragma unroll
          for (int n = 0; n < kAhead; ++n) v[n] = value_fragment<FP8>(values, n);
        };
        read_first();
        const bool clean = partial_tile<TREE, kKeys>(s, (walk.tile + i) * kKeys), beyond = __builtin_amdgcn_readfirstlane(marked) == i;
        if (beyond || clean) {
          if (beyond) {
            __syncthreads();  // (5)
#pragma unroll
            for (int r = 0; r < kGroups; ++r) {
              const f32x2 k = *reinterpret_cast<const f32x2*>(exchange + kMaxima + 8 * (16 * r + c));
              const float m_new = moved(m[r], fmaxf(k[0], k[1]));
              const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - m_new);
#pragma unroll
              for (int n = 0; n < 8; ++n) scale_in_place(acc[r][n], alpha);
              m[r] = m_new;
            }
            __syncthreads();  // (6)
          }
          if (clean) clean_tile<FP8>(kt, w, lane);
          read_first();
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const bf16x8 now = v[n % kAhead];
#pragma unroll
          for (int r = 0; r < kGroups; ++r) acc[r][n] = mfma16(now, weight[r], acc[r][n]);
          if (n + kAhead < 8) v[n % kAhead] = value_fragment<FP8>(values, n + kAhead);
          if (more && n < Loads::kLoads) loads.issue(n, lane);
          if (more && n == 7 && Loads::kLoads > 8) loads.issue(8, lane);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (more) next_page = page_at(p, table, key + kKeys, last);
      };
      int i = 0;
      for (; i + kRing - 1 < n_tiles; ++i) add(i, std::true_type{});
      for (; i < n_tiles; ++i) add(i, std::false_type{});
      __syncthreads();  // (7)
      __syncthreads();  // (8) the sums are there
#pragma unroll
      for (int r = 0; r < kGroups; ++r) {
        const f32x2 k = *reinterpret_cast<const f32x2*>(exchange + kMaxima + 8 * (16 * r + c));
        store_row<kM>(p, walk, acc[r], m[r], k[0] + k[1], r, w, lane);
      }
    }
    walk.leave_join(p);
  } while (walk.next(p));
}

}  // namespace

void launch_latent_wide(const LatentAttnParams& p, bool fp8, bool tree, int groups, hipStream_t s) {
  if (fp8 && tree) latent_attn_wide_kernel<true, true><<<groups, kThreads, 0, s>>>(p);
  else if (fp8) latent_attn_wide_kernel<true, false><<<groups, kThreads, 0, s>>>(p);
  else if (tree) latent_attn_wide_kernel<false, true><<<groups, kThreads, 0, s>>>(p);
  else latent_attn_wide_kernel<false, false><<<groups, kThreads, 0, s>>>(p);
}

}  // namespace pith
