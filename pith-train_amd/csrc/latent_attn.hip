// Attention of new tokens to the rows of a latent cache (see latent_attn.h for the work list): up to 16 query rows a sequence, the workspace and the join.
//
//   S = kappa (Q_latent C^T + Q_pe P^T),  O = softmax(S) C
//
// The 32 rows of a tile come in once (36 KB as bf16, 20 KB as e4m3) and are used twice, as keys and as values, by 16 query rows: 30 (54) flop a byte,
// far below what the matrix cores need, so the kernel is a stream of cache rows with everything else behind it. Rows are moved global -> LDS by direct
// loads, a row an instruction (bf16) or two (e4m3), eight rows a wave, all from one page, into a ring of two tiles (e4m3: three).
// Two workgroups of four wavefronts share a compute unit. A tile is a chain of phases that wait for one another (scores, exchange, softmax, result,
// requests), and two workgroups that are in different ones fill each other's gaps; one workgroup of eight waves with tiles of 64 keys took 7400
// cycles a tile however fast the rows came.
// Products are 16x16x32 with the query row as the result's column, so a lane owns one row: operand A is 16 keys (scores) or 16 features, read transposed
// (result); operand B the queries (in registers for the whole walk) or the weights.
//   scores   wave w: keys 16 (w & 1) .. of the tile against half w >> 1 of the 576 features; the halves meet in LDS
//   softmax  every wave for itself, on the sums of all keys in the order in which the second product contracts them (eight a lane: cheaper than another
//            exchange and barrier)
//   result   wave w: features 128 w ..
// Every fragment of a tile is read from LDS once for its keys and once for its values.
// The weights go into the second product as bf16, which is what the matrix cores take beside a cache of bf16 (or e4m3, widened exactly): half a step, 2^-8, of
// each, while their sum is of the unrounded ones. With e4m3 a weight is rounded once, when its row's scale is in it.
// Kernel trace, median (least): 32 sequences of up to 8192 rows, 16 heads 38.6 (36.0) us and 6.8 for the join, 171 MB in 44.7 us a call; 8 of up to 131072 e4m3 rows
// 128 (105) and 9, 536 MB in 112 us a call (outside the profiler, with the join: 4.8 TB/s); one of 517 rows 7.4 (7.1) and 4.2. Memory bounds the first two, the
// chain from work list to first tile the last.
#include "latent_attn.h"

namespace pith {
namespace {

constexpr int kThreads = 256, kM = 16, kKeys = 32, kStart = 3, kLeast = 1;

// Scores [2 halves][16 rows][32 keys] fp32: piece k (16 bytes) of a row lies at k ^ (row % 8), so that sixteen rows of 128 bytes read or written at one
// piece spread over all banks.
constexpr int kExchangeBytes = 2 * kM * kKeys * 4;
__device__ __forceinline__ int exchange_at(int row, int piece) { return row * (kKeys * 4) + ((piece ^ (row & 7)) << 4); }

// Scores of 16 keys against the query rows: STEPS times 64 latent features, then with_pe the 64 rotary ones. `at` is the place of the lane's first piece
// (its row, piece g of the swizzled 256 bytes) of the tile; piece 4 k + g lies at ^ (64 k), on whole addresses, as tiles and rows are multiples of 256 bytes.
template <bool FP8, int STEPS, int Q>
__device__ __forceinline__ f32x4 score(const char* tile, int at, int pe_at, bool with_pe, f32x4 scale, const bf16x8 (&q)[Q]) {
  const uint32_t first = lds_address(tile) + at, pe_first = lds_address(tile) + pe_at;
  f32x4 s = {};
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    bf16x8 k0, k1;
    if constexpr (FP8) {  // sixteen features a lane: two steps
      const u32x4 raw = *lds_at<u32x4>((first ^ (64 * (i & 3))) + 256 * (i >> 2));
      k0 = widen(raw[0], raw[1]);
      k1 = widen(raw[2], raw[3]);
    } else {
      k0 = *lds_at<bf16x8>((first ^ (128 * (i & 1))) + 256 * (i >> 1));
      k1 = *lds_at<bf16x8>((first ^ (128 * (i & 1) + 64)) + 256 * (i >> 1));
    }
    s = mfma16(k0, q[2 * i], s);
    s = mfma16(k1, q[2 * i + 1], s);
  }
  if constexpr (FP8) s *= scale;
  if (with_pe) {
    s = mfma16(*lds_at<bf16x8>(pe_first), q[Q - 2], s);
    s = mfma16(*lds_at<bf16x8>(pe_first ^ 64), q[Q - 1], s);
  }
  return s;
}

template <bool FP8, bool TREE>
__global__ __launch_bounds__(kThreads, 2) void latent_attn_kernel(LatentAttnParams p) {
  using T = LatentTile<FP8, kKeys>;
  using Loads = TileLoads<FP8, kKeys>;
  constexpr int kRing = FP8 ? 3 : 2;
  constexpr int kSteps = 4;          // of 64 latent features, in each half
  constexpr int Q = 2 * kSteps + 2;  // query fragments, the last two rotary (of the second half)
  __shared__ __attribute__((aligned(1024))) char lds[kRing * T::kBytes + kExchangeBytes];
  char* const exchange = lds + kRing * T::kBytes;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int kg = wave & 1, half = wave >> 1;
  Walk<kM, kKeys, kStart, kLeast> walk;
  if (!walk.start(p, lane)) return;

  const int key_row = 16 * kg + c;  // the key this lane brings
  const int key_at = key_row * T::kLatentRow + half * (T::kLatentRow / 2) + ((g ^ row_swizzle(key_row)) << 4);
  const int pe_at = T::kPe + pe_row(key_row) * 256 + (((8 * ((key_row >> 2) & 1) + g) ^ pe_swizzle(pe_row(key_row))) << 4);
  const int value_at = value_place<FP8>(wave, c, g);
  do {
    const SeqWork& s = walk.s;
    const int n_tiles = walk.n_tiles(), last = max(s.len - 1, 0);
    const int row = walk.block * kM + min(c, walk.rows(p) - 1);
    const ScalarTable table = (ScalarTable)(uintptr_t)(p.table + walk.b * p.table_rs);
    f32x4 acc[8] = {};
    float m = -INFINITY, l = 0.f;  // reference and sum (this lane's keys) of the row

    __syncthreads();  // the ring's slots and the exchange are free: every wave is through with the segment before
    const int key16 = walk.tile * kKeys + 16 * (wave >> 1);  // this wave's sixteen of the first tile
    const auto request = [&](int i) __attribute__((always_inline)) {
      const int key = key16 + i * kKeys;
      Loads(p, page_at(p, table, key, last), key, last, lds + i * T::kBytes, wave).issue_all(lane);
    };
    bf16x8 q[Q];
    char* const staged = lds + T::kBytes;  // the slots behind the first tile's
    stage_queries<kM>(p, walk, staged, wave, lane);
    request(0);
    int next_page = page_at(p, table, key16 + kRing * kKeys, last);
    wait_loads<Loads::kLoads>();  // the queries, of the waves that brought some
    __syncthreads();
    read_query<FP8, kM>(staged, c, half * (kLatent / 2), g, q);
    __syncthreads();
#pragma unroll 1
    for (int i = 1; i < min(kRing, n_tiles); ++i) request(i);
    int slot = 0;
    for (int i = 0; i < n_tiles; ++i) {
      const int key0 = (walk.tile + i) * kKeys;
      // the tiles behind this one, up to a whole ring less one, stay in flight
      const int later = min(kRing - 1, n_tiles - 1 - i);
      if (later == 2) wait_loads<2 * Loads::kLoads>();
      else if (later == 1) wait_loads<Loads::kLoads>();
      else wait_loads<0>();
      __syncthreads();
      char* const kt = lds + slot * T::kBytes;
      const bool partial = partial_tile<TREE, kKeys>(s, key0);
      {
        f32x4 sc = {};
        if constexpr (FP8) sc = *reinterpret_cast<const f32x4*>(kt + T::kScale + (16 * kg + 4 * g) * 4);
        *reinterpret_cast<f32x4*>(exchange + exchange_at(half * kM + c, 4 * kg + g)) = score<FP8, kSteps>(kt, key_at, pe_at, half == 1, sc, q);
      }
      __syncthreads();
      if (partial) clean_tile<FP8>(kt, wave, lane);
      float y[8];
      {
        const auto sum = [&](int piece) { return *reinterpret_cast<const f32x4*>(exchange + exchange_at(c, piece)) + *reinterpret_cast<const f32x4*>(exchange + exchange_at(kM + c, piece)); };
        const f32x4 lo = sum(2 * g), hi = sum(2 * g + 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = lo[e] * p.kappa, y[4 + e] = hi[e] * p.kappa;
      }
      if (partial) mask_scores<TREE, 8>(p, s, y, row / p.H, key0 + 8 * g);
      float top = y[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, y[e]);
      if (__any(top > m + kSlack)) {  // (the same for all waves: they hold the same scores)
        const float m_new = moved(m, quad_max(top));
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
        l *= alpha;
#pragma unroll
        for (int n = 0; n < 8; ++n) scale_in_place(acc[n], alpha);
        m = m_new;
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = __builtin_amdgcn_exp2f(y[e] - ref);
        l += y[e];
      }
      if constexpr (FP8) {
        const f32x4* const k = reinterpret_cast<const f32x4*>(kt + T::kScale + 8 * g * 4);
        const f32x4 s0 = k[0], s1 = k[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = scaled(y[e], s0[e]), y[4 + e] = scaled(y[4 + e], s1[e]);
      }
      const bf16x8 weight = to_bf16x8(y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]);  // keys 8 g + e
#pragma unroll
      for (int n = 0; n < 8; ++n) acc[n] = mfma16(value_fragment<FP8>(lds_address(kt) + value_at, n), weight, acc[n]);

      if (i + kRing < n_tiles) {
        __syncthreads();  // nobody reads this tile any more: its slot is asked to be filled before the next tile is waited for
        const int key = key16 + (i + kRing) * kKeys;
        Loads(p, next_page, key, last, kt, wave).issue_all(lane);
        next_page = page_at(p, table, key + kKeys, last);
      }
      slot = slot + 1 == kRing ? 0 : slot + 1;
    }
    store_row<kM>(p, walk, acc, m, quad_sum(l), 0, wave, lane);
    walk.leave_join(p);
  } while (walk.next(p));
}

constexpr int kJoinThreads = 512;
constexpr int kMaxGroups = 512;  // workgroups of the attention kernel, at most: kMaxGroups + 1 parts of a row block

// Joins the parts of a row block: o = sum_i w_i O_i / sum_i w_i l_i, w_i = 2^(m_i - max m). blockIdx.x: row block; blockIdx.y: group of 16 rows of it,
// and which `vectors` of its 32 result vectors (part_at). The weights of the rows are formed first, in one pass over their references and sums, so that
// the loads of the sums over the parts do not wait for one another (the first of them are on their way by then); where a workgroup has fewer vectors than
// waves, several waves take every other part and add up in LDS. 17 MB of parts: 6.5 us, 33 MB: 9.6; parts of one row block: 4.2, two latencies and a launch.
template <int M>
__global__ __launch_bounds__(kJoinThreads) void latent_join_kernel(LatentAttnParams p, int vectors) {
  constexpr int kWaves = kJoinThreads / 64;
  constexpr int kPerRow = kJoinThreads / 16;                     // threads that form the weights of a row
  __shared__ __attribute__((aligned(16))) f32x4 sum_o[kJoinThreads];
  __shared__ float weights[16][kMaxGroups + 1];
  __shared__ float inverse[16];  // of the rows' sums (0: nothing seen)
  const int items = *p.items;
  const LatentJoin join = p.joins[blockIdx.x];  // (beyond `items` it is whatever the workspace held)
  const int shares = kLatent / 16 / vectors, r = blockIdx.y / shares;
  if ((int)blockIdx.x >= items || join.first == join.last || 16 * r >= join.rows) return;
  const int n = min(join.last / 2 - join.first / 2 + 1, kMaxGroups + 1);  // parts: the first slot, then the even ones up to the last
  const auto slot = [&](int i) { return (int64_t)(i == 0 ? join.first : 2 * (join.first / 2 + i)); };
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15;
  const int mine = wave % vectors, group = wave / vectors, groups = kWaves / vectors;
  const int vector = blockIdx.y % shares * vectors + mine;
  const auto part = [&](int i) { return *reinterpret_cast<const f32x4*>(p.parts + part_at<M>(slot(i), r, vector, lane)); };
  f32x4 x[4];  // the first ones are on their way while the weights are formed (those behind the last one: that one, not used)
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = part(min(group + k * groups, n - 1));
  {
    const int row = threadIdx.x / kPerRow, u = threadIdx.x % kPerRow;
    const auto stat = [&](int i) { return p.stats[slot(i) * M + 16 * r + row]; };
    const float2 one = u < n ? stat(u) : make_float2(-INFINITY, 0.f);  // (most often the thread's only one)
    float top = one.x;
    for (int i = u + kPerRow; i < n; i += kPerRow) {
      const float m = stat(i).x;
      weights[row][i] = m;
      top = fmaxf(top, m);
    }
#pragma unroll
    for (int d = 1; d < kPerRow; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float ref = top == -INFINITY ? 0.f : top, w = __builtin_amdgcn_exp2f(one.x - ref);
    float sum = w * one.y;
    if (u < n) weights[row][u] = w;
    for (int i = u + kPerRow; i < n; i += kPerRow) {
      const float w = __builtin_amdgcn_exp2f(weights[row][i] - ref);
      weights[row][i] = w;
      sum += w * stat(i).y;
    }
#pragma unroll
    for (int d = 1; d < kPerRow; d <<= 1) sum += __shfl_xor(sum, d);
    if (u == 0) {
      inverse[row] = sum == 0.f ? 0.f : 1.f / sum;
      if (blockIdx.y % shares == 0 && 16 * r + row < join.rows) {
        const int at = join.row0 + 16 * r + row, tok = at / p.H;
        p.lse[(at - tok * p.H) * p.lse_hs + tok] = sum == 0.f ? -INFINITY : ref + __builtin_amdgcn_logf(sum);
      }
    }
  }
  __syncthreads();
  f32x4 o = {};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (group + k * groups < n) o += x[k] * weights[c][group + k * groups];
  int i = group + 4 * groups;
  for (; i + 3 * groups < n; i += 4 * groups) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = part(i + k * groups);
#pragma unroll
    for (int k = 0; k < 4; ++k) o += x[k] * weights[c][i + k * groups];
  }
  for (; i < n; i += groups) o += part(i) * weights[c][i];
  if (groups > 1) {
    sum_o[threadIdx.x] = o;
    __syncthreads();
    if (group > 0) return;
    for (int k = 1; k < groups; ++k) o += sum_o[64 * (k * vectors + mine) + lane];
  }
  if (16 * r + c >= join.rows) return;
  const int at = join.row0 + 16 * r + c, tok = at / p.H, head = at - tok * p.H;
  o = inverse[c] == 0.f ? f32x4{} : o * inverse[c];
  *reinterpret_cast<u32x2*>(p.o + (int64_t)tok * p.o_ts + head * p.o_hs + 16 * vector + 4 * (lane >> 4)) =
      u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

template <int M>
void launch_join(const LatentAttnParams& p, int vectors, hipStream_t s) {
  const dim3 grid(p.max_items, M / 16 * (kLatent / 16 / vectors));
  latent_join_kernel<M><<<grid, kJoinThreads, 0, s>>>(p, vectors);
}

struct LatentPlan {
  int rows;        // of a workgroup: 16 or 64
  int groups;      // workgroups of the attention kernel, a multiple of 8
  int max_items;   // row blocks at most
  int join_vectors;  // of a workgroup of the join, see there
  int64_t joins_at, stats_at, parts_at, bytes;  // workspace
};

// Workgroups of the attention kernel for m rows each: two a compute unit, or one.
int groups_of(int m) {
  const int units = (m == kM ? 2 : 1) * compute_units_or_default() & ~7;
  return units < 8 ? 8 : units > kMaxGroups ? kMaxGroups : units;
}

LatentPlan plan_of(const pith_latent_attn_args* a) {
  LatentPlan pl = {};
  const int64_t rows = a->T * a->H;
  // Blocks of 64 rows where sequences bring more than 16, unless the work list is short even with full page tables: two tiles a compute unit. In us (kernel +
  // join), 16 / 64 rows: 32 sequences of 4096 rows, 16 query rows each 29.4 + 5.9 / 35.1 + 5.1, 32 rows 36.8 + 5.5 / 35.3 + 6.0, 48 rows 73.3 + 6.2 /
  // 34.8 + 6.6; 4 sequences of 1500 rows, 64 query rows each 13.8 + 5.6 / 17.1 + 5.1, 128 rows (e4m3) 17.5 + 5.2 / 18.6 + 4.9.
  const int64_t sequences = a->B < a->T ? a->B : a->T, blocks = (rows + kWideRows - 1) / kWideRows;
  const int64_t tiles = (blocks > sequences ? blocks : sequences) * ((a->table_width * a->cache.page_size + kKeys - 1) / kKeys);
  pl.rows = rows <= kM * a->B || tiles <= 2 * compute_units_or_default() ? kM : kWideRows;
  pl.groups = groups_of(pl.rows);
  const auto items = [&](int m) { return (rows + m - 1) / m + (a->B < a->T ? a->B : a->T); };
  pl.max_items = (int)items(pl.rows);
  pl.join_vectors = 8;  // a vector a wave, or fewer where there are few row blocks
  while (pl.join_vectors > 1 && pl.max_items * (pl.rows / 16) * (kLatent / 16 / pl.join_vectors) < 512) pl.join_vectors /= 2;
  // Laid out for whichever kernel needs more: who keeps a workspace from call to call keeps one size.
  const auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  const int64_t slot_rows = 2 * std::max<int64_t>(groups_of(kM) * kM, groups_of(kWideRows) * kWideRows);
  pl.joins_at = 256;
  pl.stats_at = pl.joins_at + up(items(kM) * (int64_t)sizeof(LatentJoin));
  pl.parts_at = pl.stats_at + up(slot_rows * (int64_t)sizeof(float2));
  pl.bytes = pl.parts_at + slot_rows * kLatent * 4;
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
  if (items > 1 << 22 || items * (most / kKeys + 1) > 0x7fffffff - 65536) return fail(PITH_ERR_UNSUPPORTED, "%s: too many row blocks for page tables of that width: call it with fewer tokens at a time", who);
  return PITH_OK;
}

void launch_narrow(const LatentAttnParams& p, bool fp8, bool tree, int groups, hipStream_t s) {
  if (fp8 && tree) latent_attn_kernel<true, true><<<groups, kThreads, 0, s>>>(p);
  else if (fp8) latent_attn_kernel<true, false><<<groups, kThreads, 0, s>>>(p);
  else if (tree) latent_attn_kernel<false, true><<<groups, kThreads, 0, s>>>(p);
  else latent_attn_kernel<false, false><<<groups, kThreads, 0, s>>>(p);
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int64_t pith_latent_attn_workspace_bytes(const pith_latent_attn_args* a) {
  if (check_attn(a, "pith_latent_attn_workspace_bytes") != PITH_OK || a->T == 0 || a->B == 0) return 0;
  return plan_of(a).bytes;
}

extern "C" int pith_latent_attn_rows(const pith_latent_attn_args* a) {
  if (check_attn(a, "pith_latent_attn_rows") != PITH_OK || a->T == 0 || a->B == 0) return 0;
  return plan_of(a).rows;
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
  p.joins = (LatentJoin*)(ws + pl.joins_at);
  p.stats = (float2*)(ws + pl.stats_at);
  p.parts = (float*)(ws + pl.parts_at);
  p.max_items = pl.max_items;
  const bool fp8 = a->cache.dtype == PITH_FP8_E4M3, tree = a->tree_mask != nullptr;
  hipStream_t s = (hipStream_t)stream;
  begin_launch();
  if (pl.rows == kM) {
    launch_narrow(p, fp8, tree, pl.groups, s);
    launch_join<kM>(p, pl.join_vectors, s);
  } else {
    launch_latent_wide(p, fp8, tree, pl.groups, s);
    launch_join<kWideRows>(p, pl.join_vectors, s);
  }
  return check_launch(who);
}
