// Attention of new tokens to the rows of a latent cache, 64 query rows to a workgroup (see latent_attn.h for the work list, latent_attn.hip for the rest):
// sequences that bring more than 16 rows, by their heads or by several tokens.
//
// With 64 rows the products of a tile (64 keys: 8.9 Mflop, 2200 cycles of a compute unit's matrix cores) and its way through the address unit (72 KB at 64
// bytes a cycle: 1150) are of one size, so the work is kept off both: one workgroup of eight waves holds a compute unit, and every tile that it fetches
// serves all 64 rows. The queries stay in registers: wave w scores keys 16 (w & 3) .. of a tile against all 576 features of rows 32 (w >> 2) .. + 31 (144
// registers), and adds features 64 w .. to the results of all 64 rows (64 registers). Each key fragment is read from LDS twice, each value fragment
// once; the weights go through LDS (8 KB).
// Weights are formed against a reference of each row that all waves know from earlier tiles; only a score beyond its slack makes them meet (two barriers
// more) to move it. So a tile has two barriers: its arrival, and the weights. The loads of the next tile into the other slot stand one by one between
// the score products: issued together they take 1200 to 1600 cycles in which nothing else goes on.
#include "latent_attn.h"

namespace pith {
namespace {

constexpr int kThreads = 512, kM = kWideRows, kKeys = kWideKeys, kGroups = kM / 16;

// Weights [64 rows][64 keys] bf16, piece k (16 bytes) of a row at k ^ (row % 8); maxima (or sums) [64 rows][4 key groups] fp32; the stamp of the tile whose
// scores went beyond their slack.
constexpr int kMaxima = kM * kKeys * 2, kStamp = kMaxima + kM * 16, kExchangeBytes = kStamp + 16;
__device__ __forceinline__ int weight_at(int row, int piece) { return row * (kKeys * 2) + ((piece ^ (row & 7)) << 4); }

template <bool FP8, bool TREE>
__global__ __launch_bounds__(kThreads, 2) void latent_attn_wide_kernel(LatentAttnParams p) {
  using T = LatentTile<FP8, kKeys>;
  constexpr int kRing = FP8 ? 3 : 2;
  constexpr int J = 2;               // groups of 16 rows that a wave scores
  constexpr int kSteps = 8;          // of 64 latent features
  constexpr int Q = 2 * kSteps + 2;  // query fragments, the last two rotary
  __shared__ __attribute__((aligned(1024))) char lds[kRing * T::kBytes + kExchangeBytes];
  char* const exchange = lds + kRing * T::kBytes;
  int* const stamp = reinterpret_cast<int*>(exchange + kStamp);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave & 3, set = wave >> 2;
  Walk<kM, kKeys> walk;
  if (!walk.start(p, threadIdx.x & 63)) return;

  do {
    const SeqWork& s = walk.s;
    const int n_tiles = walk.n_tiles(), last = max(s.len - 1, 0);
    const ScalarTable table = (ScalarTable)(uintptr_t)(p.table + walk.b * p.table_rs);
    f32x4 acc[kGroups][4] = {};
    float m[kGroups], l[J];  // references of the lane's row of every group, sums (this lane's keys) of those it scores
#pragma unroll
    for (int r = 0; r < kGroups; ++r) m[r] = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) l[j] = 0.f;

    __syncthreads();  // the ring's slots and the exchange are free: every wave is through with the segment before
    if (threadIdx.x == 0) *stamp = 0;
    const int key16 = walk.tile * kKeys + 16 * (wave >> 1);  // this wave's sixteen of the first tile
    const int lane = lane_here();
    const auto request = [&](int i) __attribute__((always_inline)) {
      const int key = key16 + i * kKeys;
      TileLoads<FP8, kKeys>(p, page_of(p, table, key, last), key, last, lds + i * T::kBytes, wave).issue_all(lane);
    };
    bf16x8 q[J][Q];
    char* const staged = lds + T::kBytes;  // the slots behind the first tile's
    static_assert((kRing - 1) * T::kBytes >= LatentTile<false, kM>::kBytes, "the queries are staged in what the first tile leaves of the ring");
    stage_queries<kM>(p, walk, staged, wave, lane);
    request(0);
    int next_page = page_of(p, table, key16 + (kRing - 1) * kKeys, last);
    wait_loads<T::kLoads>();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < J; ++j) read_query<FP8, kM>(staged, 16 * (J * set + j) + (lane & 15), 0, lane >> 4, q[j]);
    __syncthreads();
    if (kRing > 2 && n_tiles > 1) request(1);
    int slot = 0;
    for (int i = 0; i < n_tiles; ++i) {
      const int key0 = (walk.tile + i) * kKeys;
      if (kRing == 2 || i + 1 >= n_tiles) wait_loads<0>();
      else wait_loads<(kRing - 2) * T::kLoads>();
      __syncthreads();
      char* const kt = lds + slot * T::kBytes;
      int into = slot + kRing - 1;
      into = into >= kRing ? into - kRing : into;
      slot = slot + 1 == kRing ? 0 : slot + 1;
      const bool partial = partial_tile<TREE, kKeys>(s, key0);
      // What the lane's number gives is formed anew in every tile: kept across the loop it would be spilled.
      const int ln = lane_here();
      const int c = ln & 15, g = ln >> 4;

      f32x4 x[J], sc = {};
      {
        const int key_row = 16 * kg + c;  // the key this lane brings
        const int key_at = key_row * T::kLatentRow + ((g ^ tile_swizzle(key_row)) << 4);
        const int pe_at = T::kPe + pe_row(key_row) * 256 + (((8 * ((key_row >> 2) & 1) + g) ^ pe_swizzle(pe_row(key_row))) << 4);
        if constexpr (FP8) sc = *reinterpret_cast<const f32x4*>(kt + T::kScale + (16 * kg + 4 * g) * 4);
        if (i + kRing - 1 < n_tiles) {
          const int key = key16 + (i + kRing - 1) * kKeys;
          const TileLoads<FP8, kKeys> loads(p, next_page, key, last, lds + into * T::kBytes, wave);
          score<FP8, J, kSteps>(kt, key_at, pe_at, true, sc, q, x, [&](int step) __attribute__((always_inline)) {
            if (2 * step < T::kLoads) loads.issue(2 * step, ln);
            if (2 * step + 1 < T::kLoads) loads.issue(2 * step + 1, ln);
          });
          next_page = page_of(p, table, key + kKeys, last);
        } else {
          score<FP8, J, kSteps>(kt, key_at, pe_at, true, sc, q, x, [](int) {});
        }
      }
      // weights against the references as they are, and whether they will do
      bool beyond = false;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        x[j] *= p.kappa;
        if (partial) mask_scores<TREE, 4>(p, s, x[j], (walk.block * kM + min(16 * (J * set + j) + c, walk.rows(p) - 1)) / p.H, key0 + 16 * kg + 4 * g);
        const float mine = set ? m[J + j] : m[j];
        beyond |= fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])) > mine + kSlack;
      }
      const auto leave_weights = [&](float (&sum)[J]) __attribute__((always_inline)) {  // and what they add to the sums
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float mine = set ? m[J + j] : m[j], ref = mine == -INFINITY ? 0.f : mine;
          f32x4 w;
#pragma unroll
          for (int v = 0; v < 4; ++v) w[v] = __builtin_amdgcn_exp2f(x[j][v] - ref);
          sum[j] = (w[0] + w[1]) + (w[2] + w[3]);
          if constexpr (FP8) {
#pragma unroll
            for (int v = 0; v < 4; ++v) w[v] = scaled(w[v], sc[v]);
          }
          *reinterpret_cast<u32x2*>(exchange + weight_at(16 * (J * set + j) + c, 2 * kg + (g >> 1)) + 8 * (g & 1)) = u32x2{pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])};
        }
      };
      float sum[J];
      leave_weights(sum);
      if (__any(beyond) && ln == 0) *stamp = i + 1;
      __syncthreads();
      if (__builtin_amdgcn_readfirstlane(*stamp) == i + 1) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float top = quad_max(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
          if (g == 0) *reinterpret_cast<float*>(exchange + kMaxima + 16 * (16 * (J * set + j) + c) + 4 * kg) = top;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kGroups; ++r) {
          const f32x4 k = *reinterpret_cast<const f32x4*>(exchange + kMaxima + 16 * (16 * r + c));
          const float m_new = fmaxf(fmaxf(fmaxf(k[0], k[1]), fmaxf(k[2], k[3])), m[r]);
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - m_new);
          if (r / J == set) l[r % J] *= alpha;
#pragma unroll
          for (int n = 0; n < 4; ++n) scale_in_place(acc[r][n], alpha);
          m[r] = m_new;
        }
        leave_weights(sum);
        __syncthreads();
      }
#pragma unroll
      for (int j = 0; j < J; ++j) l[j] += sum[j];
      if (partial && (TREE || s.n > 1)) {
        clean_tile<FP8, kKeys, kThreads>(kt);
        __syncthreads();
      }
      const uint32_t values = lds_address(kt) + value_place<FP8, 64>(wave, c, g);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        bf16x8 weight[kGroups];  // keys 32 ks + 8 g + e of the lane's row of each group
#pragma unroll
        for (int r = 0; r < kGroups; ++r) weight[r] = *reinterpret_cast<const bf16x8*>(exchange + weight_at(16 * r + c, 4 * ks + g));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const bf16x8 v = value_fragment<FP8>(values + 32 * ks * T::kLatentRow, n);
#pragma unroll
          for (int r = 0; r < kGroups; ++r) acc[r][n] = mfma16(v, weight[r], acc[r][n]);
        }
      }
    }

    const int ln = lane_here(), c = ln & 15, g = ln >> 4;
    __syncthreads();  // the last maxima have been read
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float part = quad_sum(l[j]);
      if (g == 0) *reinterpret_cast<float*>(exchange + kMaxima + 16 * (16 * (J * set + j) + c) + 4 * kg) = part;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kGroups; ++r) {
      const f32x4 k = *reinterpret_cast<const f32x4*>(exchange + kMaxima + 16 * (16 * r + c));
      store_row<FP8, kM>(p, walk, acc[r], m[r], (k[0] + k[1]) + (k[2] + k[3]), r, wave, ln);
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
