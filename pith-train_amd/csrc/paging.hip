// The bookkeeping of a step: token offsets, positions and slots of new rows, pages out of a pool and back into it (include/pith_kv.h).
//
// Everything is prefix sums over the requests: offsets are sums of the counts; pages that ended requests return go behind the pool's at sums of what they
// held; pages that are taken come off its top at sums of what is needed. A request is served if what is needed up to it and it included does not exceed the
// pool, or it needs nothing: sums only grow, so the served ones that need pages are a beginning of the list, and the order decides, not the schedule.
// One workgroup does that; up to 8192 tokens are its work too, more go to a second launch. All of it is latency: a step of 32 requests moves 1 KB. Up to 64
// requests are a lane each and need no barrier for their sums; up to 1024 are a thread each, with four barriers (three more where pages come back) and sums of 32 bits. us of a call, launch
// included: 32 requests of a token each 7.1, 423 8.7 (12.2 in the loop for any number, whose sums have 64 bits), 1000 11.8 (16.2); 16 prompts, 16384 tokens, 10.
#include "cache_attn.h"
#include "pith_kv.h"

namespace pith {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kInOne = kThreads;  // requests whose sums stay in LDS

struct PlanParams {
  const int32_t* counts;
  const int32_t* lengths;
  int32_t* table;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* cu_q;
  int64_t* positions;
  int64_t* slots;
  int32_t* granted;
  int32_t* lengths_out;
  int32_t* free_count_out;
  int64_t T, table_rs, table_width, pool;
  int B, page_shift;
  // workspace of the two-launch form: what the tokens need to know of their requests, the pool's top before pages were taken
  struct Request* requests;
  int64_t* top;
};

// A request as its tokens see it.
struct Request {
  int32_t length;  // rows before the step
  int32_t served;
  int64_t taken;   // pages that requests in front of it take
};

// Inclusive sums over the workgroup, and the sum of all.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* waves, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the sums of the scan before have been read
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int64_t s = waves[w];
    before += w < wave ? s : 0;
    total += s;
  }
  return before + x;
}

// The same of 32 bits, with room of its own for every call: one barrier.
__device__ __forceinline__ int block_scan(int x, int* waves) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  x = wave_scan(x);
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  const int sums = wave_scan(lane < wave ? waves[lane] : 0);
  return x + __builtin_amdgcn_readlane(sums, 63);
}

// Position and slot of token t; the first row of a page that was taken brings it into the table. `cu(i)`, `request(i)`: of request i.
template <typename C, typename R>
__device__ __forceinline__ void place_token(const PlanParams& p, int64_t t, int64_t top, const C& cu, const R& request) {
  int64_t position = 0, slot = -1;
  if (t < cu(p.B)) {
    int lo = 0, hi = p.B - 1;  // the last request whose offset is at or below t (one that has tokens: those behind it begin further on)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu(mid) <= t) lo = mid;
      else hi = mid - 1;
    }
    const Request r = request(lo);
    position = r.length + (t - cu(lo));
    if (r.served) {
      const int64_t index = position >> p.page_shift, held = ((int64_t)r.length + (1 << p.page_shift) - 1) >> p.page_shift;
      int32_t* const entry = p.table + lo * p.table_rs + index;
      const int64_t in_page = position & ((1 << p.page_shift) - 1);
      int32_t page;
      if (index < held) {
        page = *entry;
      } else {
        page = p.free_pages[top - 1 - (r.taken + index - held)];
        if (in_page == 0) *entry = page;
      }
      slot = ((int64_t)page << p.page_shift) + in_page;
    }
  }
  p.positions[t] = position;
  p.slots[t] = slot;
}

// Any number of requests; the tokens are for the next launch.
__global__ __launch_bounds__(kThreads) void plan_kernel(PlanParams p) {
  __shared__ int64_t waves[kWaves];
  __shared__ int64_t base[kInOne];
  __shared__ int32_t held_of[kInOne];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t page_size = (int64_t)1 << p.page_shift, most = p.table_width << p.page_shift;
  const auto length_of = [&](int i) { return (int32_t)min(max((int64_t)p.lengths[i], (int64_t)0), most); };
  const auto pages_of = [&](int64_t rows) { return (rows + page_size - 1) >> p.page_shift; };
  const int64_t had = min(max((int64_t)p.free_count[0], (int64_t)0), p.pool);

  // pages that come back
  int64_t back = 0, total;
  for (int i0 = 0; i0 < p.B; i0 += kInOne) {
    const int i = i0 + tid;
    const int64_t held = i < p.B && p.counts[i] < 0 ? pages_of(length_of(i)) : 0;
    const int64_t upto = block_scan(held, waves, total);
    if (total == 0) continue;  // (uniform)
    base[tid] = had + back + upto - held;
    held_of[tid] = (int32_t)held;
    __syncthreads();
    for (int r = wave; r < min(kInOne, p.B - i0); r += kWaves) {  // a wave each
      const int n = held_of[r];
      const int32_t* const row = p.table + (i0 + r) * p.table_rs;
      for (int k = lane; k < n; k += 64)
        if (base[r] + k < p.pool) p.free_pages[base[r] + k] = row[k];
    }
    back += total;
  }
  const int64_t top = min(had + back, p.pool);
  __syncthreads();  // what was laid on the pool is there

  // rows and pages of the others
  int64_t rows_before = 0, need_before = 0;
  int64_t taken = 0;  // this thread's: what requests up to its last served one take
  for (int i0 = 0; i0 < p.B; i0 += kInOne) {
    const int i = i0 + tid;
    const bool some = i < p.B;
    const int32_t count = some ? p.counts[i] : 0;
    const int32_t length = some ? length_of(i) : 0;
    const int64_t upto = block_scan(max(count, 0), waves, total) + rows_before;
    const int64_t first = min(upto - max(count, 0), p.T), last = min(upto, p.T), rows = last - first;
    rows_before += total;
    const bool fits = count >= 0 && length + rows <= most;
    const int64_t need = fits ? pages_of(length + rows) - pages_of(length) : 0;
    const int64_t needed = block_scan(need, waves, total) + need_before;
    need_before += total;
    const bool served = fits && (need == 0 || needed <= top);
    if (served && need > 0) taken = needed;
    if (some) {
      p.granted[i] = served ? (int32_t)rows : 0;
      p.lengths_out[i] = count < 0 ? 0 : length + (served ? (int32_t)rows : 0);
      p.cu_q[i + 1] = (int32_t)last;
      p.requests[i] = Request{length, served, needed - need};
    }
  }
  if (tid == 0) p.cu_q[0] = 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) taken = max(taken, (int64_t)__shfl_xor(taken, d));
  __syncthreads();
  if (lane == 0) waves[wave] = taken;
  __syncthreads();
  if (tid == 0) {
    for (int w = 0; w < kWaves; ++w) taken = max(taken, waves[w]);
    p.free_count_out[0] = (int32_t)(top - taken);
    *p.top = top;
  }
}

// Up to kInOne requests, a thread each, and up to kTokensInOne tokens in the same launch, or up to kTokensIn32 in the next: 32 bits hold all sums but those of the pages that
// come back.
constexpr int64_t kTokensInOne = 8192, kTokensIn32 = 1 << 20;
__global__ __launch_bounds__(kThreads) void plan_some_kernel(PlanParams p) {
  __shared__ int64_t back_sums[kWaves];
  __shared__ int64_t base[kInOne];
  __shared__ int32_t held_of[kInOne], cu_of[kInOne + 1], row_sums[kWaves], page_sums[kWaves], most_taken[kWaves];
  __shared__ Request request_of[kInOne];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int page = 1 << p.page_shift, most = (int)(p.table_width << p.page_shift), tokens = (int)p.T;
  const bool some = tid < p.B;
  const int count = some ? p.counts[tid] : 0;
  const int length = some ? min(max(p.lengths[tid], 0), most) : 0;
  const int64_t had = min(max((int64_t)p.free_count[0], (int64_t)0), p.pool);
  const auto pages_of = [&](int rows) { return (int)(((unsigned)rows + page - 1) >> p.page_shift); };
  const int held = pages_of(length);

  int64_t back = 0;
  if (__syncthreads_or(count < 0)) {  // (the barrier is also for those that have yet to read what is written below)
    const int64_t mine = count < 0 ? held : 0;
    base[tid] = had + block_scan(mine, back_sums, back) - mine;
    held_of[tid] = (int)mine;
    __syncthreads();
    for (int r = wave; r < p.B; r += kWaves) {  // a wave each
      const int n = held_of[r];
      for (int k = lane; k < n; k += 64)
        if (base[r] + k < p.pool) p.free_pages[base[r] + k] = p.table[r * p.table_rs + k];
    }
  }
  const int64_t top = min(had + back, p.pool);

  const int wanted = min(max(count, 0), tokens);
  const int upto = block_scan(wanted, row_sums), first = min(upto - wanted, tokens), last = min(upto, tokens), rows = last - first;
  const bool fits = count >= 0 && rows <= most - length;
  const int need = fits ? pages_of(length + rows) - held : 0;
  const int needed = block_scan(need, page_sums);
  const bool served = fits && (need == 0 || needed <= top);
  const int taken = wave_scan_max(served && need > 0 ? needed : 0);
  if (lane == 63) most_taken[wave] = taken;
  if (some) {
    p.granted[tid] = served ? rows : 0;
    p.lengths_out[tid] = count < 0 ? 0 : length + (served ? rows : 0);
    p.cu_q[tid + 1] = cu_of[tid + 1] = last;
    request_of[tid] = Request{length, served, needed - need};
  }
  if (tid == 0) p.cu_q[0] = cu_of[0] = 0;
  __syncthreads();  // (and what was laid on the pool is there)
  if (wave == 0) {
    const int all = wave_scan_max(lane < kWaves ? most_taken[lane] : 0);
    if (lane == 63) p.free_count_out[0] = (int32_t)(top - all);
  }
  if (p.requests) {  // (the tokens are for the next launch)
    if (some) p.requests[tid] = request_of[tid];
    if (tid == 0) *p.top = top;
    return;
  }
  for (int t = tid; t < tokens; t += kThreads)
    place_token(p, t, top, [&](int i) { return (int64_t)cu_of[i]; }, [&](int i) { return request_of[i]; });
}

__global__ __launch_bounds__(256) void place_kernel(PlanParams p) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t < p.T) place_token(p, t, *p.top, [&](int i) { return (int64_t)p.cu_q[i]; }, [&](int i) { return p.requests[i]; });
}

// The same for up to 64 requests, a lane each: every wave forms all sums by itself, and looks a token's request up among its lanes. No LDS; a barrier behind
// what all waves read and the first writes, and another where pages come back.
__global__ __launch_bounds__(kThreads) void plan_few_kernel(PlanParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int page = 1 << p.page_shift;
  const bool some = lane < p.B;
  const int most = (int)(p.table_width << p.page_shift), tokens = (int)p.T;
  const int count = some ? p.counts[lane] : 0;
  const int length = some ? min(max(p.lengths[lane], 0), most) : 0;
  const int64_t had = min(max((int64_t)p.free_count[0], (int64_t)0), p.pool);
  const auto pages_of = [&](int rows) { return (int)(((unsigned)rows + page - 1) >> p.page_shift); };
  const int held = pages_of(length);

  int64_t back = 0;
  __syncthreads();  // every wave has read what the first will write
  if (__any(count < 0)) {
    int64_t upto = count < 0 ? held : 0;
    const int64_t mine = upto;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
    back = __shfl(upto, 63);
    for (int r = wave; r < p.B; r += waves) {
      const int n = (int)__shfl(mine, r);
      const int64_t base = had + __shfl(upto - mine, r);
      for (int k = lane; k < n; k += 64)
        if (base + k < p.pool) p.free_pages[base + k] = p.table[r * p.table_rs + k];
    }
    __syncthreads();  // what was laid on the pool is there
  }
  const int64_t top = min(had + back, p.pool);

  const int wanted = min(max(count, 0), tokens);  // (their sum is below 2^31: few tokens, or 2^24 at most)
  const int upto = wave_scan(wanted), first = min(upto - wanted, tokens), last = min(upto, tokens), rows = last - first;
  const bool fits = count >= 0 && rows <= most - length;
  const int need = fits ? pages_of(length + rows) - held : 0;
  const int needed = wave_scan(need), taken = needed - need;
  const bool served = fits && (need == 0 || needed <= top);
  if (wave == 0) {
    if (some) {
      p.granted[lane] = served ? rows : 0;
      p.lengths_out[lane] = count < 0 ? 0 : length + (served ? rows : 0);
      p.cu_q[lane + 1] = last;
    }
    const int all = wave_scan_max(served && need > 0 ? needed : 0);
    if (lane == 63) {
      p.cu_q[0] = 0;
      p.free_count_out[0] = (int32_t)(top - all);
    }
    if (p.requests) {  // (the tokens are for the next launch)
      if (some) p.requests[lane] = Request{length, served, taken};
      if (lane == 63) *p.top = top;
    }
  }
  if (p.requests) return;
  const int end = __builtin_amdgcn_readlane(last, 63);
  for (int t0 = wave * 64; t0 < tokens; t0 += 64 * waves) {
    const int t = t0 + lane;
    int r = 0;  // requests that end at or before t
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
      if (__shfl(last, r + d - 1) <= t) r += d;
    r = min(r, 63);
    const int before = __shfl(length, r), into = t - __shfl(first, r);
    const int position = (int)((unsigned)before + (unsigned)into);  // (of a request that is served: below 2^31)
    const int index = position >> p.page_shift, in_page = position & (page - 1);
    const int beyond = index - __shfl(held, r);
    const int64_t at = top - 1 - __shfl(taken, r) - beyond;
    int64_t slot = -1;
    if (__shfl((int)served, r) && t < end) {
      int32_t* const entry = p.table + r * p.table_rs + index;
      const int32_t number = beyond < 0 ? *entry : p.free_pages[at];
      if (beyond >= 0 && in_page == 0) *entry = number;
      slot = ((int64_t)number << p.page_shift) + in_page;
    }
    if (t < tokens) {
      p.positions[t] = t < end ? (int64_t)before + into : 0;
      p.slots[t] = slot;
    }
  }
}

bool in_one(const pith_plan_step_args* a) { return a->B <= kInOne && a->T <= kTokensInOne; }

int check_plan(const pith_plan_step_args* a, const char* who) {
  if (!a) return fail(PITH_ERR_NULL_POINTER, "%s: args is NULL", who);
  if (a->B < 0 || a->T < 0 || a->B > 1 << 20 || a->T > 0x7fffffff || a->table_width < 0 || a->pool_size < 0 || a->pool_size > 0x7fffffff)
    return fail(PITH_ERR_BAD_SHAPE, "%s: B = %lld (at most 2^20), T = %lld, table_width = %lld, pool_size = %lld (below 2^31)", who, (long long)a->B, (long long)a->T,
                (long long)a->table_width, (long long)a->pool_size);
  if (a->page_size < 16 || a->page_size > 65536 || (a->page_size & (a->page_size - 1)))
    return fail(PITH_ERR_BAD_SHAPE, "%s: page size %lld is not a power of two from 16 to 65536", who, (long long)a->page_size);
  if (a->table_width > 0x7fffffff / a->page_size) return fail(PITH_ERR_UNSUPPORTED, "%s: page tables of 2^31 rows or more", who);
  return PITH_OK;
}

}  // namespace
}  // namespace pith

using namespace pith;

extern "C" int pith_kv_version(void) { return PITH_KV_VERSION; }

extern "C" int64_t pith_plan_step_workspace_bytes(const pith_plan_step_args* a) {
  if (check_plan(a, "pith_plan_step_workspace_bytes") != PITH_OK || in_one(a)) return 0;
  return (16 + a->B * (int64_t)sizeof(Request) + 15) & ~(int64_t)15;
}

extern "C" int pith_plan_step(const pith_plan_step_args* a, pith_stream_t stream) {
  const char* who = "pith_plan_step";
  if (const int rc = check_plan(a, who)) return rc;
  const bool one = in_one(a);
  if (!a->cu_q || !a->free_count || !a->free_count_out || (a->T > 0 && (!a->position_ids || !a->slots)) || (a->pool_size > 0 && !a->free_pages) ||
      (a->B > 0 && (!a->counts || !a->lengths || !a->granted || !a->lengths_out || (!a->page_table && a->table_width > 0))) || (!one && !a->workspace))
    return fail(PITH_ERR_NULL_POINTER, "%s: a required pointer is NULL", who);
  if (a->B > 1 && a->table_rs < a->table_width) return fail(PITH_ERR_BAD_SHAPE, "%s: rows of the page table overlap", who);
  const auto off = [](const void* x, unsigned n) { return (uintptr_t)x % n != 0; };
  if (off(a->counts, 4) || off(a->lengths, 4) || off(a->page_table, 4) || off(a->free_pages, 4) || off(a->free_count, 4) || off(a->cu_q, 4) || off(a->granted, 4) ||
      off(a->lengths_out, 4) || off(a->free_count_out, 4) || off(a->position_ids, 8) || off(a->slots, 8) || off(a->workspace, 16))
    return fail(PITH_ERR_MISALIGNED, "%s: arrays need the alignment of their elements, the workspace 16 bytes", who);
  if (!one && a->workspace_bytes < pith_plan_step_workspace_bytes(a))
    return fail(PITH_ERR_BAD_SHAPE, "%s: the workspace has %lld bytes, %lld are needed", who, (long long)a->workspace_bytes, (long long)pith_plan_step_workspace_bytes(a));
  PlanParams p = {};
  p.counts = a->counts; p.lengths = a->lengths; p.table = a->page_table; p.free_pages = a->free_pages; p.free_count = a->free_count;
  p.cu_q = a->cu_q; p.positions = a->position_ids; p.slots = a->slots; p.granted = a->granted; p.lengths_out = a->lengths_out; p.free_count_out = a->free_count_out;
  p.T = a->T; p.table_rs = a->B > 1 ? a->table_rs : 0; p.table_width = a->table_width; p.pool = a->pool_size;
  p.B = (int)a->B; p.page_shift = __builtin_ctzll((unsigned long long)a->page_size);
  hipStream_t s = (hipStream_t)stream;
  begin_launch();
  if (one && a->B <= 64) {
    const int64_t threads = (a->T + 63) & ~(int64_t)63;
    plan_few_kernel<<<1, (unsigned)(threads < 64 ? 64 : threads > kThreads ? kThreads : threads), 0, s>>>(p);
  } else if (one) {
    plan_some_kernel<<<1, kThreads, 0, s>>>(p);
  } else {
    p.top = (int64_t*)a->workspace;
    p.requests = (Request*)((char*)a->workspace + 16);
    if (a->B <= 64 && a->T <= 1 << 24) plan_few_kernel<<<1, 256, 0, s>>>(p);
    else if (a->B <= kInOne && a->T <= kTokensIn32) plan_some_kernel<<<1, kThreads, 0, s>>>(p);
    else plan_kernel<<<1, kThreads, 0, s>>>(p);
    if (a->T > 0) place_kernel<<<(unsigned)((a->T + 255) / 256), 256, 0, s>>>(p);
  }
  return check_launch(who);
}
