// Which pages of a long cache a token attends to (include/pith_kv.h): a bound of q . k over every page from the least and largest values of its key
// features, then the pages with the largest bounds in the order of the sequence.
//
//   score(page) = max over the heads of the group of sum_d max(q_d least_d, q_d largest_d)
//
// A choice must not depend on the order of a sum, or the same scores would choose differently elsewhere: products of two bf16 values are exact in fp32, and
// their sum in fp64 loses nothing that a rounding to fp32 would show. Scores are kept as integers that sort like them, NaN above all.
#include "kv_common.h"

namespace pith {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kChunk = 64;  // pages of a workgroup that scores, one a lane

struct KVSelectParams {
  const __bf16 *q, *bounds;
  const int32_t *table, *lengths, *cu_q;
  int32_t *table_out, *lengths_out;
  uint32_t* keys;  // [T * heads][row]
  int64_t q_ts, q_hs, table_rs, bounds_ps, row;
  int T, B, heads, group, pages, page_shift, table_width, keep, chunks;
};

// Rows that token t sees, 0 for one that is nobody's.
__device__ __forceinline__ int visible_rows(const KVSelectParams& p, int t, int seq) {
  const int length = min(max(p.lengths[seq], 0), p.table_width << p.page_shift);
  if (!p.cu_q) return length;
  return t < p.cu_q[p.B] ? min(max(length - p.cu_q[seq + 1] + t + 1, 0), length) : 0;
}

__device__ __forceinline__ float nan_max(float a, float b) { return b > a || b != b ? b : a; }

__device__ __forceinline__ uint32_t sort_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Scores of 64 pages of a token and key-value head: a page a lane, out of LDS (rows of 4 D bytes, piece (16 bytes) k of row r at k ^ r % (D / 4), so that
// the lanes' reads of one piece spread over the banks); a wave takes two heads of the group at a time.
template <int D>
__global__ __launch_bounds__(kThreads) void kv_score_kernel(KVSelectParams p) {
  constexpr int kPieces = D / 4;  // of a page's bounds: D least, D largest
  __shared__ __attribute__((aligned(16))) char rows[kChunk * kPieces * 16];
  __shared__ float best[kWaves][kChunk];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = blockIdx.x % p.chunks, item = blockIdx.x / p.chunks;  // (token, head)
  const int t = item / p.heads, head = item - t * p.heads;
  const int seq = sequence_of(p.cu_q, p.B, t, lane);
  const int visible = visible_rows(p, t, seq);
  const int pages = (visible + (1 << p.page_shift) - 1) >> p.page_shift;
  const int first = chunk * kChunk, n = min(pages - 1 - first, kChunk);  // (the token's own page is not scored)
  if (pages <= p.keep || n <= 0) return;
  const int32_t* const table = p.table + seq * p.table_rs + first;
#pragma unroll
  for (int i = threadIdx.x; i < kChunk * kPieces; i += kThreads) {
    const int r = i / kPieces, piece = i % kPieces;
    const int64_t page = safe_page(table[min(r, n - 1)], p.pages);
    *reinterpret_cast<u32x4*>(rows + r * (kPieces * 16) + ((piece ^ (r % kPieces)) << 4)) =
        *reinterpret_cast<const u32x4*>(p.bounds + page * p.bounds_ps + (int64_t)head * (2 * D) + 8 * piece);
  }
  __syncthreads();
  float top = -INFINITY;
  const char* const mine = rows + lane * (kPieces * 16);
  for (int h = 2 * wave; h < p.group; h += 2 * kWaves) {
    const __bf16* const q0 = p.q + t * p.q_ts + (int64_t)(head * p.group + h) * p.q_hs;
    const __bf16* const q1 = p.q + t * p.q_ts + (int64_t)(head * p.group + min(h + 1, p.group - 1)) * p.q_hs;
    double s0 = 0., s1 = 0.;
#pragma unroll 2
    for (int d = 0; d < D; d += 8) {
      const u32x4 lo = *reinterpret_cast<const u32x4*>(mine + (((d / 8) ^ (lane % kPieces)) << 4));
      const u32x4 hi = *reinterpret_cast<const u32x4*>(mine + (((d / 8 + D / 8) ^ (lane % kPieces)) << 4));
      const u32x4 a = *reinterpret_cast<const u32x4*>(q0 + d), b = *reinterpret_cast<const u32x4*>(q1 + d);  // (wave-uniform)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const auto value = [&](const u32x4& x) { return e & 1 ? bf16hi_to_f32(x[e >> 1]) : bf16lo_to_f32(x[e >> 1]); };
        const float x0 = value(a), x1 = value(b), least = value(lo), largest = value(hi);
        s0 += (double)__builtin_elementwise_maximum(x0 * least, x0 * largest);  // (NaN stays)
        s1 += (double)__builtin_elementwise_maximum(x1 * least, x1 * largest);
      }
    }
    top = nan_max(nan_max(top, (float)s0), (float)s1);
  }
  best[wave][lane] = top;
  __syncthreads();
  if (wave == 0 && lane < n) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = nan_max(top, best[w][lane]);
    p.keys[item * p.row + first + lane] = sort_key(top);
  }
}

// Inclusive sums over the workgroup.
__device__ __forceinline__ int block_scan(int x, int* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  for (int w = 0; w < wave; ++w) x += waves[w];
  return x;
}

constexpr int kInLds = 8192;  // scores that are kept in LDS

// The keep - 1 largest of a token's and head's scores: their least one digit by digit (8 bits, from the top, a histogram each), then every thread counts those
// above it and equal to it in a stretch of the sequence, and writes its own behind those of the stretches in front of it.
__global__ __launch_bounds__(kThreads) void kv_pick_kernel(KVSelectParams p) {
  __shared__ uint32_t kept[kInLds];
  __shared__ int histogram[256];
  __shared__ int waves[kWaves], digit, rest;
  const int tid = threadIdx.x, lane = tid & 63;
  const int item = blockIdx.x, t = item / p.heads;
  const int seq = sequence_of(p.cu_q, p.B, t, lane);
  const int visible = visible_rows(p, t, seq);
  const int pages = (visible + (1 << p.page_shift) - 1) >> p.page_shift;
  const int n = min(pages, p.keep);
  const int32_t* const table = p.table + seq * p.table_rs;
  int32_t* const out = p.table_out + (int64_t)item * p.keep;
  if (tid == 0) p.lengths_out[item] = visible - ((pages - n) << p.page_shift);
  for (int i = n + tid; i < p.keep; i += kThreads) out[i] = -1;
  if (pages <= p.keep) {
    for (int i = tid; i < n; i += kThreads) out[i] = table[i];
    return;
  }
  if (tid == 0) out[n - 1] = table[pages - 1];
  if (n == 1) return;
  const uint32_t* const keys = p.keys + item * p.row;
  const int scored = pages - 1;
  const bool in_lds = scored <= kInLds;
  if (in_lds)
    for (int i = tid; i < scored; i += kThreads) kept[i] = keys[i];
  const auto key = [&](int i) { return in_lds ? kept[i] : keys[i]; };
  uint32_t least = 0;  // of the largest ones, as far as its digits are known
  int want = n - 1;    // of those that begin with these digits
  for (int shift = 24; shift >= 0; shift -= 8) {
    histogram[tid] = 0;
    __syncthreads();
    for (int i = tid; i < scored; i += kThreads) {
      const uint32_t k = key(i);
      if (shift == 24 || (k ^ least) >> (shift + 8) == 0) atomicAdd(&histogram[(k >> shift) & 255], 1);
    }
    __syncthreads();
    const int mine = histogram[255 - tid], upto = block_scan(mine, waves);
    if (upto >= want && upto - mine < want) digit = 255 - tid, rest = want - (upto - mine);
    __syncthreads();
    least |= (uint32_t)digit << shift;
    want = rest;
  }
  const int each = (scored + kThreads - 1) / kThreads, from = min(tid * each, scored), to = min(from + each, scored);
  int above = 0, equal = 0;
  for (int i = from; i < to; ++i) {
    const uint32_t k = key(i);
    above += k > least;
    equal += k == least;
  }
  const int equals_before = block_scan(equal, waves) - equal;  // of equal ones the first `want` count
  const int take = min(max(want - equals_before, 0), equal);
  int at = block_scan(above + take, waves) - (above + take), equals = 0;
  for (int i = from; i < to; ++i) {
    const uint32_t k = key(i);
    if (k > least || (k == least && equals++ < take)) out[at++] = table[i];
  }
}

int check_select(const pith_kv_select_args* a, const char* who) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (const int rc = check_pages(a->pages, a->page_size, a->heads, a->dim, who)) return rc;
  if (const int rc = check_table(a->T, a->B, a->heads, a->table_width, a->page_size, !a->cu_q, who)) return rc;
  if (a->H < 1 || a->H > 1024 || a->H % a->heads) return fail(PITH_ERR_BAD_SHAPE, "%s: %lld query heads (at most 1024) of %lld key-value heads", who, (long long)a->H, (long long)a->heads);
  if (a->keep < 1 || a->keep > 1 << 20) return fail(PITH_ERR_BAD_SHAPE, "%s: keep = %lld pages (1 to 2^20)", who, (long long)a->keep);
  if (a->T * a->heads > 0x7fffffff / ((a->table_width + kChunk - 1) / kChunk + 1) || a->T * a->heads > (int64_t)1 << 24)
    return fail(PITH_ERR_UNSUPPORTED, "%s: too many tokens for page tables of that width: call it with fewer at a time", who);
  return PITH_OK;
}

int64_t chunks_of(const pith_kv_select_args* a) { return (a->table_width + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int64_t pith_kv_select_workspace_bytes(const pith_kv_select_args* a) {
  if (check_select(a, "pith_kv_select_workspace_bytes") != PITH_OK || a->B == 0) return 0;
  return a->T * a->heads * chunks_of(a) * kChunk * 4;
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
  p.table_out = a->table_out; p.lengths_out = a->lengths_out; p.keys = (uint32_t*)a->workspace;
  p.q_ts = a->q_ts; p.q_hs = a->q_hs; p.table_rs = a->B > 1 ? a->table_rs : 0; p.bounds_ps = a->pages > 1 ? a->bounds_ps : 0;
  p.chunks = (int)chunks_of(a); p.row = (int64_t)p.chunks * kChunk;
  p.T = (int)a->T; p.B = (int)a->B; p.heads = (int)a->heads; p.group = (int)(a->H / a->heads);
  p.pages = (int)a->pages; p.page_shift = __builtin_ctzll((unsigned long long)a->page_size); p.table_width = (int)a->table_width; p.keep = (int)a->keep;
  hipStream_t s = (hipStream_t)stream;
  begin_launch();
  const unsigned items = (unsigned)(a->T * a->heads);
  if (a->keep > 1 && a->table_width > a->keep) {  // (else nothing is scored)
    if (a->dim == 128) kv_score_kernel<128><<<items * (unsigned)p.chunks, kThreads, 0, s>>>(p);
    else kv_score_kernel<64><<<items * (unsigned)p.chunks, kThreads, 0, s>>>(p);
  }
  kv_pick_kernel<<<items, kThreads, 0, s>>>(p);
  return check_launch(who);
}
