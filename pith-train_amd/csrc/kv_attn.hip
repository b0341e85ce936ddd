// Attention of new tokens to the rows of a key-value cache: heads of 128 features, the join, the plan of a call (see kv_attn.h; heads of 64: kv_attn_d64.hip).
#include "kv_attn.h"

#include <algorithm>

namespace pith {

void launch_kv_attn_d128(const KVAttnParams& p, bool fp8, int row_groups, int workgroups, hipStream_t s) { launch_kv_attn<128>(p, fp8, row_groups, workgroups, s); }

namespace {

constexpr int kJoinThreads = 512, kJoinRows = 4;
constexpr int kMaxGroups = 512;  // workgroups of the attention kernel, at most, where row blocks are cut: kMaxGroups + 1 parts of one

// Joins the parts of a row block: o = sum_i w_i O_i / sum_i w_i l_i, w_i = 2^(m_i - max m). blockIdx.x: entry of the joins, blockIdx.y: four rows of it. A wave forms
// the weights of a row; then groups of threads, a piece of four features each, take every so many-th part and meet in LDS.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void kv_join_kernel(KVAttnParams p, int m) {
  constexpr int kPieces = D / 4, kEach = kJoinRows * kPieces, kGroups = kJoinThreads / kEach;
  __shared__ f32x4 sums[kJoinThreads];
  __shared__ float weights[kJoinRows][kMaxGroups + 1];
  __shared__ float inverse[kJoinRows];  // of the rows' sums (0: nothing seen)
  const int row0 = kJoinRows * blockIdx.y;
  const int items = *p.items;
  const KVJoin join = p.joins[blockIdx.x];  // (beyond `items` it is whatever the workspace held)
  if ((int)blockIdx.x >= items || join.parts == 1 || row0 >= join.rows) return;
  const int n = min(join.parts, kMaxGroups + 1);
  const auto slot = [&](int i) { return (int64_t)(i == 0 ? join.first : join.second + (i - 1) * join.stride); };
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = threadIdx.x / kEach, row = threadIdx.x % kEach / kPieces, piece = threadIdx.x % kPieces;
  const auto part = [&](int i) { return *reinterpret_cast<const f32x4*>(p.results + (slot(i) * m + row0 + row) * D + 4 * piece); };
  f32x4 x[4];  // the first ones are on their way while the weights are formed (those behind the last one: that one, not used)
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = part(min(group + k * kGroups, n - 1));
  const auto place = [&](int r, int& h, int64_t& t) {  // of a row of the row block
    const int at = join.row0 + r, tok = at / p.group;
    h = join.head * p.group + at - tok * p.group;
    t = join.tok0 + tok;
  };
  if (wave < kJoinRows) {
    const auto stat = [&](int i) { return p.stats[slot(i) * m + row0 + wave]; };
    float top = -INFINITY, sum = 0.f;
    for (int i = lane; i < n; i += 64) top = fmaxf(top, stat(i).x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float ref = top == -INFINITY ? 0.f : top;
    for (int i = lane; i < n; i += 64) {
      const float2 s = stat(i);
      const float w = __builtin_amdgcn_exp2f(s.x - ref);
      weights[wave][i] = w;
      sum += w * s.y;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) {
      inverse[wave] = sum == 0.f ? 0.f : 1.f / sum;
      if (row0 + wave < join.rows) {
        int h;
        int64_t t;
        place(row0 + wave, h, t);
        p.lse[h * p.lse_hs + t] = sum == 0.f ? -INFINITY : ref + __builtin_amdgcn_logf(sum);
      }
    }
  }
  __syncthreads();
  f32x4 o = {};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (group + k * kGroups < n) o += x[k] * weights[row][group + k * kGroups];
  int i = group + 4 * kGroups;
  for (; i + 3 * kGroups < n; i += 4 * kGroups) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = part(i + k * kGroups);
#pragma unroll
    for (int k = 0; k < 4; ++k) o += x[k] * weights[row][i + k * kGroups];
  }
  for (; i < n; i += kGroups) o += part(i) * weights[row][i];
  sums[threadIdx.x] = o;
  __syncthreads();
  if (group > 0 || row0 + row >= join.rows) return;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) o += sums[k * kEach + threadIdx.x];
  o = inverse[row] == 0.f ? f32x4{} : o * inverse[row];
  int h;
  int64_t t;
  place(row0 + row, h, t);
  *reinterpret_cast<u32x2*>(p.o + t * p.o_ts + h * p.o_hs + 4 * piece) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

struct KVPlan {
  int row_groups;  // of 16 query rows, to a row block
  int workgroups;  // a multiple of 8
  int whole;       // steps of the longest row block where none is cut, else 0
  int parts;       // of every row block, where all are cut alike (into two or more), else 0
  bool by_range;   // joins are the workgroups'
  int64_t max_items;  // row blocks, or joins
  int64_t joins_at, stats_at, results_at, bytes;  // workspace
};

KVPlan plan_of(const pith_kv_attn_args* a) {
  KVPlan pl = {};
  const int units = std::max(compute_units_or_default() & ~7, 8);
  const int64_t group = a->H / a->cache.heads, rows = a->T * group;  // rows of a key-value head
  const int64_t steps = (a->table_width * a->cache.page_size + kStepKeys - 1) / kStepKeys, sequences = std::min(a->B, a->T);
  const auto items = [&](int64_t m) { return ((rows + m - 1) / m + sequences) * a->cache.heads; };
  // Rows of a row block. Fewer bytes and products with more of them, but every workgroup begins and ends with them more slowly, and rows that are not there are
  // computed all the same: so 16 for sequences of no more, and while with blocks of 16 and full page tables a compute unit has few steps (32) and few row blocks
  // (2.5; heads of 64, which have half the bytes and products, twice of both). us at 16 / 32 rows, heads of 32 / 4: 8 tokens, e4m3, 8 x 4096
  // rows (20 steps) 24 / 26, bf16, 16 x 2048 (20) 23 / 24, 8 x 8192 (40) 38 / 33, 16 x 8192 (80) 114 / 53; 16 tokens, e4m3, 16 x 2048 (36) 41 / 37; 2 tokens, 32 x 8192
  // 75 / 76; heads of 64 / 4, 8 tokens, 35 x 131 22 / 19 (few steps, but 3 row blocks); of 16 / 2 with 64 features, 14 tokens, 75 x 1530 (56 steps, 4.7 row blocks) 44 / 49.
  // And 64 for bf16 heads of 128 where that makes the row blocks fewer by a quarter and keys and values are about as much as the last-level cache holds, or more: 8 tokens,
  // 32 x 8192 (540 MB) 115 at 32 rows and 92 at 64, 18, 55 x 1771 (200 MB) 91 / 76, 6, 64 x 2048 (270 MB) 65 / 65, but 8 tokens, 8 x 8192 (130 MB) 30 / 33, 64 x 1024 (130 MB)
  // 43 / 53, 512 behind 8192 rows (17 MB) 109 / 119. (64 rows of e4m3 or of heads of 64 lose, or gain 7 % at most: 16 tokens, 16 x 8192 e4m3 77 / 80, 8, 32 x 8192, 64
  // features 62 / 58.)
  const double work = (double)items(16) * steps / units, bytes = (double)sequences * steps * kStepKeys * a->cache.heads * 512;
  const int64_t each = (rows + sequences - 1) / sequences;
  const bool small = work * a->cache.dim <= 32 * 128 && 2 * items(16) * a->cache.dim <= 5 * units * 128;
  const bool fewer = 4 * ((each + 63) / 64) <= 3 * ((each + 31) / 32);
  if (rows <= 16 * a->B || small) pl.row_groups = 1;
  else pl.row_groups = a->cache.dtype == PITH_BF16 && a->cache.dim == 128 && fewer && bytes >= (192 << 20) ? 4 : 2;
  const int64_t m = 16 * pl.row_groups;
  const int per_unit = pl.row_groups <= 2 ? 2 : 1;  // workgroups (KVRing)
  pl.max_items = items(m);
  // No row block is cut where that would gain less than the join's launch costs (4 us), as long as all of them begin at once, and long ones do not share a compute unit: one
  // sequence of 517 rows, 4 heads, 8.8 us whole and 10.6 cut (with weights of 8 bits), 8 x 1024 rows, 8 tokens 12 / 17, 23 x 71 rows (460 row blocks) 10 / 13; but 64 x 900 (384) 28 / 25, 86 x 2
  // (688) 14.6 / 13.1.
  bool whole = (steps * pl.row_groups <= 8 && pl.max_items <= units) || (steps * pl.row_groups <= 2 && pl.max_items <= per_unit * units);
  pl.workgroups = std::min(per_unit * units, kMaxGroups);
  if (a->head_tables) {
    pl.max_items = (group + m - 1) / m * a->cache.heads * a->B;
    pl.parts = (int)std::min(std::max<int64_t>(pl.workgroups / pl.max_items, 1), steps);
    pl.workgroups = (int)((pl.max_items * pl.parts + 7) & ~(int64_t)7);
    whole = whole || pl.parts == 1;
  }
  if (whole) {
    pl.whole = (int)steps;
    pl.parts = 0;
    pl.workgroups = (int)((pl.max_items + 7) & ~(int64_t)7);
    pl.bytes = 256;
    return pl;
  }
  // A join for each workgroup where the row blocks are more: of 4096 (1024 sequences of up to 200 rows, e4m3) 512 at most are cut, 87 us with a join for each row block,
  // 79 so; 8 prompts of 512 tokens 119 / 106.
  pl.by_range = !pl.parts && pl.max_items > pl.workgroups;
  if (pl.by_range) pl.max_items = pl.workgroups;
  const auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  const int64_t slot_rows = (pl.parts ? 1 : 2) * (int64_t)pl.workgroups * m;
  pl.joins_at = 256;
  pl.stats_at = pl.joins_at + up(pl.max_items * (int64_t)sizeof(KVJoin));
  pl.results_at = pl.stats_at + up(slot_rows * (int64_t)sizeof(float2));
  pl.bytes = pl.results_at + slot_rows * a->cache.dim * 4;
  return pl;
}

int check_attn(const pith_kv_attn_args* a, const char* who) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (const int rc = check_cache(a->cache, who)) return rc;
  if (const int rc = check_table(a->T, a->B, a->cache.heads, a->table_width, a->cache.page_size, !a->cu_q, who)) return rc;
  if (a->H < 1 || a->H > 1024 || a->H % a->cache.heads)
    return fail(PITH_ERR_BAD_SHAPE, "%s: %lld query heads (at most 1024) of %lld key-value heads", who, (long long)a->H, (long long)a->cache.heads);
  // counted in 32 bits on the device: row blocks, and the steps of the whole work list
  const int64_t items = ((a->T * (a->H / a->cache.heads) + 15) / 16 + a->B) * a->cache.heads;
  if (items > 1 << 24 || a->B * a->cache.heads > 1 << 24 || items * (a->table_width * a->cache.page_size / kStepKeys + 1) > 0x7fffffff - (1 << 25))
    return fail(PITH_ERR_UNSUPPORTED, "%s: too many row blocks for page tables of that width: call it with fewer tokens at a time", who);
  if (a->head_tables && (a->tree_mask || a->cu_q)) return fail(PITH_ERR_UNSUPPORTED, "%s: tables of the heads go with one token a sequence: no cu_q, no tree_mask", who);
  return PITH_OK;
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int64_t pith_kv_attn_workspace_bytes(const pith_kv_attn_args* a) {
  if (check_attn(a, "pith_kv_attn_workspace_bytes") != PITH_OK || a->T == 0 || a->B == 0) return 0;
  return plan_of(a).bytes;
}

extern "C" int pith_kv_attn_rows(const pith_kv_attn_args* a) {
  if (check_attn(a, "pith_kv_attn_rows") != PITH_OK || a->T == 0 || a->B == 0) return 0;
  return 16 * plan_of(a).row_groups;
}

extern "C" int pith_kv_attn(const pith_kv_attn_args* a, pith_stream_t stream) {
  const char* who = "pith_kv_attn";
  if (const int rc = check_attn(a, who)) return rc;
  if (a->T == 0 || a->B == 0) return PITH_OK;
  if (!a->q || !a->lengths || !a->o || !a->lse || !a->workspace || (!a->page_table && a->table_width > 0))
    return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if (a->table_width == 0) return fail(PITH_ERR_BAD_SHAPE, "%s: an empty page table holds no rows", who);
  const int64_t dim = a->cache.dim, heads = a->cache.heads;
  if ((a->B > 1 && a->table_rs < a->table_width) || (a->head_tables && heads > 1 && a->table_hs < a->table_width) || (a->T > 1 && (a->q_ts < dim || a->o_ts < dim)) ||
      (a->H > 1 && (a->q_hs < dim || a->o_hs < dim || a->lse_hs < a->T)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: a stride is shorter than what it steps over", who);
  if (!aligned16(a->q) || !aligned16(a->o) || (a->q_ts | a->q_hs | a->o_ts | a->o_hs) % 8 || (uintptr_t)a->workspace % 256 || (uintptr_t)a->page_table % 4 ||
      (uintptr_t)a->lengths % 4 || (uintptr_t)a->cu_q % 4 || (uintptr_t)a->lse % 4 || (uintptr_t)a->tree_mask % 8)
    return fail(PITH_ERR_MISALIGNED, "%s: queries and results need 16-byte alignment and strides of multiples of 8, the workspace 256-byte alignment", who);
  const KVPlan pl = plan_of(a);
  if (a->workspace_bytes < pl.bytes) return fail(PITH_ERR_BAD_SHAPE, "%s: the workspace has %lld bytes, %lld are needed", who, (long long)a->workspace_bytes, (long long)pl.bytes);
  KVAttnParams p = {};
  p.q = (const __bf16*)a->q; p.cache = to_device(a->cache); p.table = a->page_table; p.lengths = a->lengths; p.cu_q = a->cu_q; p.tree = a->tree_mask;
  p.o = (__bf16*)a->o; p.lse = a->lse;
  p.table_rs = a->B > 1 ? a->table_rs : 0; p.table_hs = a->head_tables && heads > 1 ? a->table_hs : 0;
  p.q_ts = a->q_ts; p.q_hs = a->q_hs; p.o_ts = a->o_ts; p.o_hs = a->o_hs; p.lse_hs = a->lse_hs;
  p.T = (int)a->T; p.B = (int)a->B; p.H = (int)a->H; p.group = (int)(a->H / heads); p.table_width = (int)a->table_width;
  p.head_tables = a->head_tables ? (int)heads : 1;
  p.max_len = (int)(a->table_width * a->cache.page_size);
  p.kappa = a->scale * 1.4426950408889634f;
  p.whole = pl.whole; p.parts = pl.parts;
  char* const ws = (char*)a->workspace;
  p.items = (int*)ws;
  p.joins = (KVJoin*)(ws + pl.joins_at);
  p.stats = (float2*)(ws + pl.stats_at);
  p.results = (float*)(ws + pl.results_at);
  p.max_items = (int)pl.max_items;
  p.by_range = pl.by_range;
  hipStream_t s = (hipStream_t)stream;
  const bool fp8 = a->cache.dtype == PITH_FP8_E4M3;
  begin_launch();
  if (dim == 128) launch_kv_attn_d128(p, fp8, pl.row_groups, pl.workgroups, s);
  else launch_kv_attn_d64(p, fp8, pl.row_groups, pl.workgroups, s);
  if (!pl.whole) {
    const dim3 grid((unsigned)pl.max_items, (unsigned)(16 * pl.row_groups / kJoinRows));
    if (dim == 128) kv_join_kernel<128><<<grid, kJoinThreads, 0, s>>>(p, 16 * pl.row_groups);
    else kv_join_kernel<64><<<grid, kJoinThreads, 0, s>>>(p, 16 * pl.row_groups);
  }
  return check_launch(who);
}
