// Attention of new tokens to the rows of a latent cache (see latent_attn.h for the work list).
//
//   S = kappa (Q_latent C^T + Q_pe P^T),  O = softmax(S) C
//
// The 64 rows of a tile come in once (72 KB as bf16, 40 KB as e4m3) and are used twice, as keys and as values, by all rows of a workgroup: 30 (54)
// flop a byte with 16 query rows, where the kernel is a stream of cache rows with everything else behind it, and four times that with 64, where the
// matrix cores are as busy as the memory. One workgroup of eight wavefronts holds a compute unit: a ring of two tiles (e4m3: three) nearly fills its
// LDS. Rows are moved global -> LDS by direct loads, a row an instruction (bf16) or two (e4m3), eight rows a wave, all from one page.
// Products are 16x16x32 with the query row as the result's column, so a lane owns one row of each group of 16: operand A is 16 keys (scores) or 16
// features, read transposed (result); operand B the queries (in registers for the whole walk) or the weights.
//   16 rows  wave w scores keys 16 (w & 3) .. against half w >> 2 of the 576 features. The halves meet in LDS (8 KB), where every wave reads the sums of
//            all keys in the order in which the second product contracts them and forms the weights for itself: two barriers a tile.
//   64 rows  wave w scores keys 16 (w & 3) .. against all features of 32 rows, 32 (w >> 2) ..; the maxima of the four key groups meet in LDS (1 KB),
//            then the weights (9 KB): three barriers a tile.
// Then wave w adds features 64 w .. of all rows. Every fragment of a tile is read from LDS once (16 rows) or twice (64 rows: the keys).
#include "latent_attn.h"

namespace pith {
namespace {

constexpr int kThreads = 512;

template <bool FP8>
struct Tile {
  static constexpr int kLatentRow = FP8 ? kLatent : 2 * kLatent;  // bytes
  static constexpr int kPe = kLatentKeys * kLatentRow;            // offsets in a tile
  static constexpr int kScale = kPe + kLatentKeys * 2 * kRope;    // [64] fp32
  static constexpr int kBytes = kScale + (FP8 ? kLatentKeys * 4 : 0);
  static constexpr int kLoads = FP8 ? 6 : 9;  // direct loads of a wave
  static constexpr int kRing = FP8 ? 3 : 2;
};

// What the waves of a workgroup exchange: RG = 1 row group: scores [2 halves][16 rows][68]; RG = 4: weights [64 rows][72] bf16, maxima [64][4].
constexpr int kScoreRow = kLatentKeys + 4, kWeightRow = kLatentKeys + 8;  // the ends spread the rows over the banks
template <int RG>
constexpr int kExchangeBytes = RG == 1 ? 2 * 16 * kScoreRow * 4 : 16 * RG * (kWeightRow * 2 + 16);

// Piece (16 bytes) swizzles: piece q of a row lies at q ^ swizzle(row). Latent rows are whole multiples of 256 bytes; the low four bits of the piece
// are swizzled so that sixteen consecutive rows read at one piece hit different banks (tile_swizzle, attn_tiles.h). Rotary rows lie two to a 256-byte
// LDS row: row 8 w + i and 8 w + 4 + i (i < 4) in pieces 0-7 and 8-15 of LDS row 4 w + i, so that a wave's eight rows are one instruction.
__device__ __forceinline__ int pe_row(int row) { return ((row >> 3) << 2) | (row & 3); }
__device__ __forceinline__ int pe_swizzle(int lds_row) { return ((lds_row & 3) << 1) | ((lds_row >> 2) & 1); }

// Page of the sixteen rows from key on (a multiple of 16); rows behind the sequence's last one are read as that one.
// Read as constant memory (nobody writes tables while the kernel runs): a scalar load, which the counted waits for tiles do not see.
typedef const __attribute__((address_space(4))) int32_t* ScalarTable;
__device__ __forceinline__ int page_of(const LatentAttnParams& p, ScalarTable table, int key, int last) {
  return safe_page(table[min(key, last) >> p.cache.page_shift], p.cache.pages);
}

// Issues wave w's direct loads of a tile: rows 8 w .. 8 w + 7 of it, which are half of the sixteen from key16 = key0 + 16 (w >> 1) on.
template <bool FP8>
__device__ __forceinline__ void issue_tile(const LatentAttnParams& p, int page, int key16, int last, char* slot, int wave, int lane) {
  using T = Tile<FP8>;
  const int first = min(key16, last) & ~15;  // the page's sixteen rows
  const int in_page = first & ((1 << p.cache.page_shift) - 1);
  const int left = last - first;  // rows behind `first` that exist
  const int r0 = 8 * (wave & 1);  // of the sixteen
  const char* const base = p.cache.latent + page * p.cache.latent_ps + (int64_t)in_page * T::kLatentRow;
  char* const dst = slot + 8 * wave * T::kLatentRow;
  asm volatile("" : "+v"(lane));  // the rows' offsets are formed on the spot, not kept (and spilled) from tile to tile
  if constexpr (FP8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // two rows an instruction
      const int r = 2 * i + (lane >> 5);
      load_lds16(base, min(r0 + r, left) * T::kLatentRow + 16 * ((lane & 31) ^ tile_swizzle(8 * wave + r)), dst + 2 * i * T::kLatentRow);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      load_lds16(base + min(r0 + i, left) * T::kLatentRow, 16 * (lane ^ tile_swizzle(8 * wave + i)), dst + i * T::kLatentRow);
  }
  const int sub = lane >> 4;
  const int piece = (lane & 15) ^ pe_swizzle(4 * wave + sub);
  const char* const pe = reinterpret_cast<const char*>(p.cache.k_pe + page * p.cache.k_pe_ps + (int64_t)in_page * kRope);
  load_lds16(pe, min(r0 + 4 * (piece >> 3) + sub, left) * (2 * kRope) + 16 * (piece & 7), slot + T::kPe + wave * 1024);
  if constexpr (FP8) {
    if (lane < 8) load_lds4(p.cache.scale + page * p.cache.scale_ps + in_page + min(r0 + lane, left), slot + T::kScale + 32 * wave);
  }
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// max / sum over the four lanes c, c + 16, c + 32, c + 48 that share a query row
__device__ __forceinline__ float quad_max(float x) {
  const int i = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  return pair_max(fmaxf(__int_as_float(r[0]), __int_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
  const int i = __float_as_int(x);
  const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  return pair_sum(__int_as_float(r[0]) + __int_as_float(r[1]));
}

template <int LATER>
__device__ __forceinline__ void wait_loads() {
  static_assert(LATER < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (LATER & 15) | ((LATER >> 4) << 14));
  asm volatile("" ::: "memory");
}

// Eight e4m3 values (two words) -> bf16, exact.
__device__ __forceinline__ bf16x8 widen(uint32_t w0, uint32_t w1) {
  const bf16x2 a = fp8x2_to_bf16<false>(w0), b = fp8x2_to_bf16<true>(w0), c = fp8x2_to_bf16<false>(w1), d = fp8x2_to_bf16<true>(w1);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Scores of 16 keys against J groups of query rows: STEPS times 64 latent features, then with_pe the 64 rotary ones. `at` is the place of the lane's
// first piece (its row, piece g of the swizzled 256 bytes) of the tile; piece 4 k + g lies at ^ (64 k), as rows are multiples of 256 bytes.
template <bool FP8, int J, int STEPS, int Q>
__device__ __forceinline__ void score(const char* tile, int at, int pe_at, bool with_pe, f32x4 scale, const bf16x8 (&q)[J][Q], f32x4 (&s)[J]) {
#pragma unroll
  for (int j = 0; j < J; ++j) s[j] = f32x4{};
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    bf16x8 k0, k1;
    if constexpr (FP8) {  // sixteen features a lane: two steps
      const u32x4 raw = *reinterpret_cast<const u32x4*>(tile + (at ^ (64 * (i & 3))) + 256 * (i >> 2));
      k0 = widen(raw[0], raw[1]);
      k1 = widen(raw[2], raw[3]);
    } else {
      k0 = *reinterpret_cast<const bf16x8*>(tile + (at ^ (128 * (i & 1))) + 256 * (i >> 1));
      k1 = *reinterpret_cast<const bf16x8*>(tile + (at ^ (128 * (i & 1) + 64)) + 256 * (i >> 1));
    }
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = mfma16(k0, q[j][2 * i], s[j]);
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = mfma16(k1, q[j][2 * i + 1], s[j]);
  }
  if constexpr (FP8) {
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] *= scale;
  }
  if (with_pe) {
    const bf16x8 k0 = *reinterpret_cast<const bf16x8*>(tile + pe_at), k1 = *reinterpret_cast<const bf16x8*>(tile + (pe_at ^ 64));
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = mfma16(k0, q[j][Q - 2], s[j]);
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = mfma16(k1, q[j][Q - 1], s[j]);
  }
}

// Which feature of the wave's 64 result v of product n is in a lane of group g. Transposed reads take their columns in groups of four (bf16) or eight
// (e4m3) from wherever a lane points; as bf16 the groups of two products are dealt so that a lane's results of both are eight consecutive ones.
template <bool FP8>
__device__ __forceinline__ int feature_of(int n, int g) {
  return FP8 ? 16 * n + 4 * g : 32 * (n >> 1) + 8 * g + 4 * (n & 1);
}

// Place of the lane's transposed reads of the wave's 64 features in rows 0-31 of a tile; those of other pieces and rows are ^ and + from there.
template <bool FP8>
__device__ __forceinline__ int value_place(int wave, int c, int g) {
  const int r = 8 * g + (FP8 ? c >> 1 : c >> 2);
  const int piece = FP8 ? 4 * wave : 8 * wave + (c & 3);
  return r * Tile<FP8>::kLatentRow + ((piece ^ tile_swizzle(r)) << 4) + (FP8 ? 8 * (c & 1) : 0);
}

// Operand A of product n over keys 32 ks + 8 g + e.
template <bool FP8>
__device__ __forceinline__ bf16x8 value_fragment(const char* tile, int at, int n, int ks) {
  const char* const rows = tile + 32 * ks * Tile<FP8>::kLatentRow;
  if constexpr (FP8) {
    typedef __attribute__((ext_vector_type(2))) int i32x2;
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(rows + (at ^ (16 * n))));
    return widen((uint32_t)raw[0], (uint32_t)raw[1]);
  } else {  // four rows further on the swizzle differs in its lowest bit
    return lds_read_transposed_at(rows + (at ^ (64 * (n >> 1))) + 8 * (n & 1), rows + (at ^ (64 * (n >> 1) + 16)) + 4 * Tile<false>::kLatentRow + 8 * (n & 1));
  }
}

// Infinities and NaN of a tile's latent rows -> 0, in place, by all threads. For tiles that some rows see in part only: a row's weight of a key it does
// not see is 0, and must stay so against whatever the key holds. A row that sees such a key has a score of the same kind.
template <bool FP8>
__device__ __forceinline__ void clean_tile(char* tile) {
  for (int at = 16 * threadIdx.x; at < Tile<FP8>::kPe; at += 16 * kThreads) {
    u32x4 x = *reinterpret_cast<const u32x4*>(tile + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (FP8) {
#pragma unroll
        for (int k = 0; k < 32; k += 8)
          if (((x[e] >> k) & 0x7fu) == 0x7fu) x[e] &= ~(0xffu << k);
      } else {
        if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u;
        if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0xffffu;
      }
    }
    *reinterpret_cast<u32x4*>(tile + at) = x;
  }
}

// A weight times its row's scale; 0 stays 0, also against a scale that is not finite.
__device__ __forceinline__ float scaled(float weight, float scale) { return weight == 0.f ? 0.f : weight * scale; }

// x *= f in place: as a plain product under a branch the accumulators are copied on the other way, which doubles their registers. The compiler does not
// look into the statement for hazards: f may come from v_exp_f32 right before it (one wait state), and x from products of the tile before (two barriers
// away).
__device__ __forceinline__ void scale_in_place(f32x4& x, float f) {
  float a = x[0], b = x[1], c = x[2], d = x[3];
  asm("s_nop 1\n\tv_mul_f32 %0, %4, %0\n\tv_mul_f32 %1, %4, %1\n\tv_mul_f32 %2, %4, %2\n\tv_mul_f32 %3, %4, %3" : "+v"(a), "+v"(b), "+v"(c), "+v"(d) : "v"(f));
  x = f32x4{a, b, c, d};
}

// RG: groups of 16 query rows of a workgroup, 1 or 4.
template <bool FP8, bool TREE, int RG>
__global__ __launch_bounds__(kThreads, 2) void latent_attn_kernel(LatentAttnParams p) {
  using T = Tile<FP8>;
  constexpr int kM = 16 * RG, kRing = T::kRing;
  constexpr bool kHalves = RG == 1;          // the two sets of four waves share the features, not the rows
  constexpr int J = kHalves ? 1 : RG / 2;    // row groups that a wave scores
  constexpr int kSteps = kHalves ? 4 : 8;    // 64 latent features each
  constexpr int Q = 2 * kSteps + 2;          // query fragments, the last two rotary (halves: of the second one)
  __shared__ __attribute__((aligned(1024))) char lds[kRing * T::kBytes + kExchangeBytes<RG>];
  char* const exchange = lds + kRing * T::kBytes;
  float* const scores = reinterpret_cast<float*>(exchange);                      // RG = 1
  __bf16* const weights = reinterpret_cast<__bf16*>(exchange);                   // RG = 4
  float* const maxima = reinterpret_cast<float*>(exchange + kM * kWeightRow * 2);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave & 3, set = wave >> 2;

  // ---- the range of this workgroup: sums over the sequences, by every wave for itself. In long lists neighbours share an XCD (workgroups are
  // dealt to the eight of them in turn), whose cache then serves the row blocks of a sequence.
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
  const bool full = RG > 1 && total >= 2 * (int)gridDim.x;
  const int id = full ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x;
  const int begin = id * per, end = min(begin + per, total);  // (the host has bounded total + gridDim * min_tiles)
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
    const ScalarTable table = (ScalarTable)(uintptr_t)(p.table + b * p.table_rs);
    const int ctx = s.len - s.n;  // rows in front of the new ones (below zero only where the lengths contradict each other)
    const int last = max(s.len - 1, 0);
    const int c = lane & 15, g = lane >> 4;

    // ---- queries: features 32 st + 8 g .. of the row in step st (e4m3 keys are read 16 features at a time: steps 2 i, 2 i + 1 then contract features
    // 64 i + 16 g + {0..7, 8..15})
    bf16x8 q[J][Q];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int row = row0 + min(16 * (kHalves ? 0 : J * set + j) + c, rows - 1);
      const int tok = row / p.H, head = row - tok * p.H;
      const __bf16* ql = p.q_latent + (int64_t)(s.tok0 + tok) * p.q_ts + head * p.q_hs + (kHalves ? set * (kLatent / 2) : 0);
      const __bf16* qp = p.q_pe + (int64_t)(s.tok0 + tok) * p.q_pe_ts + head * p.q_pe_hs;
#pragma unroll
      for (int i = 0; i < Q - 2; ++i) q[j][i] = *reinterpret_cast<const bf16x8*>(ql + (FP8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g));
#pragma unroll
      for (int i = 0; i < 2; ++i) q[j][Q - 2 + i] = *reinterpret_cast<const bf16x8*>(qp + 32 * i + 8 * g);
    }

    f32x4 acc[RG][4] = {};
    float m[RG], l[J];
#pragma unroll
    for (int r = 0; r < RG; ++r) m[r] = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) l[j] = 0.f;
    // Scores of the keys that the lane's row of group j does not see -> -infinity; key_of(v): the key of score v. In the last tiles of a sequence only, so
    // what the row sees is looked up anew there.
    const auto mask = [&](auto& x, auto n_scores, int j, auto key_of) __attribute__((always_inline)) {
      const int row = row0 + min(16 * (kHalves ? 0 : J * set + j) + c, rows - 1);
      const int tok = row / p.H;
      const uint64_t word = TREE ? (uint64_t)p.tree[s.tok0 + tok] : 0;
#pragma unroll
      for (int v = 0; v < decltype(n_scores)::value; ++v) {
        const int key = key_of(v);
        bool seen = key < s.len;
        if constexpr (TREE) seen = seen && (key < ctx || (key - ctx < 64 && ((word >> ((key - ctx) & 63)) & 1)));
        else seen = seen && key <= ctx + tok;
        x[v] = seen ? x[v] : -INFINITY;
      }
    };

    __syncthreads();  // the ring's slots and the exchange are free: every wave is through with the row block before
    const int key16 = tile * kLatentKeys + 16 * (wave >> 1);  // this wave's sixteen of the first tile
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i)
      if (i < n_tiles) issue_tile<FP8>(p, page_of(p, table, key16 + i * kLatentKeys, last), key16 + i * kLatentKeys, last, lds + i * T::kBytes, wave, lane);
    int next_page = page_of(p, table, key16 + (kRing - 1) * kLatentKeys, last);
    // The queries have to be there before the walk: left to their first use, the compiler's waits for them would stand in the loop and wait for the tiles
    // in flight in every turn.
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int k = 0; k < Q; ++k) asm volatile("" : "+v"(q[j][k]));
    }
    int slot = 0;
    for (int i = 0; i < n_tiles; ++i) {
      const int key0 = (tile + i) * kLatentKeys;
      if (kRing == 2 || i + 1 >= n_tiles) wait_loads<0>();
      else wait_loads<(kRing - 2) * T::kLoads>();
      __syncthreads();
      if (i + kRing - 1 < n_tiles) {
        const int key = key16 + (i + kRing - 1) * kLatentKeys;
        int into = slot + kRing - 1;
        into = into >= kRing ? into - kRing : into;
        issue_tile<FP8>(p, next_page, key, last, lds + into * T::kBytes, wave, lane);
        next_page = page_of(p, table, key + kLatentKeys, last);
      }
      char* const kt = lds + slot * T::kBytes;
      // What the lane's number gives is formed anew in every tile of 64 rows: kept across the loop it would be spilled.
      int ln = lane;
      if constexpr (!kHalves) asm volatile("" : "+v"(ln));
      const int c = ln & 15, g = ln >> 4;
      const int key_row = 16 * kg + c;  // the key this lane brings
      const int key_at = key_row * T::kLatentRow + (kHalves ? set * (T::kLatentRow / 2) : 0) + ((g ^ tile_swizzle(key_row)) << 4);
      const int pe_at = T::kPe + pe_row(key_row) * 256 + (((8 * ((key_row >> 2) & 1) + g) ^ pe_swizzle(pe_row(key_row))) << 4);
      const int value_at = value_place<FP8>(wave, c, g);
      slot = slot + 1 == kRing ? 0 : slot + 1;
      const bool partial = key0 + kLatentKeys > ctx + (TREE ? 0 : 1);  // some row may not see all of the tile

      f32x4 sc = {};
      if constexpr (FP8) sc = *reinterpret_cast<const f32x4*>(kt + T::kScale + (16 * kg + 4 * g) * 4);
      f32x4 x[J];
      score<FP8, J, kSteps>(kt, key_at, pe_at, !kHalves || set == 1, sc, q, x);

      bf16x8 own[2];  // 16 rows: the weights of keys 32 ks + 8 g + e
      if constexpr (kHalves) {
        *reinterpret_cast<f32x4*>(scores + (set * 16 + c) * kScoreRow + 16 * kg + 4 * g) = x[0];
        __syncthreads();
        if (partial && s.n > 1) {
          clean_tile<FP8>(kt);
          __syncthreads();
        }
        float y[16];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const f32x4* const r0 = reinterpret_cast<const f32x4*>(scores + c * kScoreRow + 32 * ks + 8 * g);
          const f32x4* const r1 = reinterpret_cast<const f32x4*>(scores + (16 + c) * kScoreRow + 32 * ks + 8 * g);
          const f32x4 lo = r0[0] + r1[0], hi = r0[1] + r1[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[8 * ks + e] = lo[e] * p.kappa, y[8 * ks + 4 + e] = hi[e] * p.kappa;
        }
        if (partial) mask(y, std::integral_constant<int, 16>{}, 0, [&](int e) { return key0 + 32 * (e >> 3) + 8 * g + (e & 7); });
        float top = y[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, y[e]);
        const float m_new = fmaxf(m[0], quad_max(top));
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        if (__any(m_new > m[0])) {
          const float alpha = __builtin_amdgcn_exp2f(m[0] - ref);
          l[0] *= alpha;
#pragma unroll
          for (int n = 0; n < 4; ++n) scale_in_place(acc[0][n], alpha);
          m[0] = m_new;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          y[e] = __builtin_amdgcn_exp2f(y[e] - ref);
          l[0] += y[e];
        }
        if constexpr (FP8) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const f32x4* const k = reinterpret_cast<const f32x4*>(kt + T::kScale + (32 * ks + 8 * g) * 4);
            const f32x4 lo = k[0], hi = k[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[8 * ks + e] = scaled(y[8 * ks + e], lo[e]), y[8 * ks + 4 + e] = scaled(y[8 * ks + 4 + e], hi[e]);
          }
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          own[ks] = to_bf16x8(y[8 * ks], y[8 * ks + 1], y[8 * ks + 2], y[8 * ks + 3], y[8 * ks + 4], y[8 * ks + 5], y[8 * ks + 6], y[8 * ks + 7]);
      } else {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          x[j] *= p.kappa;
          if (partial) mask(x[j], std::integral_constant<int, 4>{}, j, [&](int v) { return key0 + 16 * kg + 4 * g + v; });
          const float top = quad_max(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));
          if (g == 0) maxima[4 * (16 * (J * set + j) + c) + kg] = top;
        }
        __syncthreads();
        if (partial && s.n > 1) clean_tile<FP8>(kt);  // (a barrier follows)
        float m_new[RG];
        bool grown = false;
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          const f32x4 k = *reinterpret_cast<const f32x4*>(maxima + 4 * (16 * r + c));
          m_new[r] = fmaxf(fmaxf(fmaxf(k[0], k[1]), fmaxf(k[2], k[3])), m[r]);
          grown |= m_new[r] > m[r];
        }
        if (__any(grown)) {
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            const float alpha = __builtin_amdgcn_exp2f(m[r] - (m_new[r] == -INFINITY ? 0.f : m_new[r]));
            if (r / J == set) l[r % J] *= alpha;
#pragma unroll
            for (int n = 0; n < 4; ++n) scale_in_place(acc[r][n], alpha);
            m[r] = m_new[r];
          }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float mine = set ? m[J + j] : m[j];
          const float ref = mine == -INFINITY ? 0.f : mine;
          f32x4 y;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            y[v] = __builtin_amdgcn_exp2f(x[j][v] - ref);
            l[j] += y[v];
          }
          if constexpr (FP8) {
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = scaled(y[v], sc[v]);
          }
          const u32x2 two = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
          *reinterpret_cast<u32x2*>(weights + (16 * (J * set + j) + c) * kWeightRow + 16 * kg + 4 * g) = two;
        }
        __syncthreads();
      }

#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        bf16x8 weight[RG];
#pragma unroll
        for (int r = 0; r < RG; ++r) weight[r] = kHalves ? own[ks] : *reinterpret_cast<const bf16x8*>(weights + (16 * r + c) * kWeightRow + 32 * ks + 8 * g);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const bf16x8 v = value_fragment<FP8>(kt, value_at, n, ks);
#pragma unroll
          for (int r = 0; r < RG; ++r) acc[r][n] = mfma16(v, weight[r], acc[r][n]);
        }
      }
    }

    // ---- the row block's result, or this part of it
    float sum[RG];  // of the lane's row of every group
    if constexpr (kHalves) {
      sum[0] = quad_sum(l[0]);
    } else {
      __syncthreads();  // the last maxima have been read
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float part = quad_sum(l[j]);
        if (g == 0) maxima[4 * (16 * (J * set + j) + c) + kg] = part;
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        const f32x4 k = *reinterpret_cast<const f32x4*>(maxima + 4 * (16 * r + c));
        sum[r] = (k[0] + k[1]) + (k[2] + k[3]);
      }
    }
    const bool whole = n_tiles == s.tiles;
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      const int row = 16 * r + c;
      if (whole) {
        if (row < rows) {
          const int tok = (row0 + row) / p.H, head = row0 + row - tok * p.H;
          const float inv = 1.f / sum[r];
          __bf16* const dst = p.o + (int64_t)(s.tok0 + tok) * p.o_ts + head * p.o_hs + 64 * wave;
#pragma unroll
          for (int n = 0; n < 4; n += 2) {
            const f32x4 a = sum[r] == 0.f ? f32x4{} : acc[r][n] * inv, d = sum[r] == 0.f ? f32x4{} : acc[r][n + 1] * inv;
            const u32x2 lo = {pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3])}, hi = {pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3])};
            if constexpr (FP8) {
              *reinterpret_cast<u32x2*>(dst + feature_of<true>(n, g)) = lo;
              *reinterpret_cast<u32x2*>(dst + feature_of<true>(n + 1, g)) = hi;
            } else {
              *reinterpret_cast<u32x4*>(dst + feature_of<false>(n, g)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
          }
          if (wave == 0 && g == 0) p.lse[head * p.lse_hs + s.tok0 + tok] = sum[r] == 0.f ? -INFINITY : m[r] + __builtin_amdgcn_logf(sum[r]);
        }
      } else if (row < rows) {
        const int64_t part = 2 * id + (at == begin ? 0 : 1);
        float* const dst = p.parts + (part * kM + row) * kLatent + 64 * wave;
#pragma unroll
        for (int n = 0; n < 4; ++n) *reinterpret_cast<f32x4*>(dst + feature_of<FP8>(n, g)) = acc[r][n];
        if (wave == 0 && g == 0) p.stats[part * kM + row] = make_float2(m[r], sum[r]);
      }
    }
    if (tile + n_tiles == s.tiles && threadIdx.x == 0 && item < p.max_items) {  // who ends a row block says where its parts lie
      const int first_tile = at + n_tiles - s.tiles;  // of the whole work list
      const int g0 = whole ? 0 : first_tile / per;
      p.joins[item] = make_int4(s.tok0 * p.H + row0, rows, whole ? 0 : 2 * g0 + (first_tile == g0 * per ? 0 : 1), whole ? 0 : 2 * id);
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

constexpr int kJoinThreads = 256;
constexpr int kMaxGroups = 1024;  // workgroups of the attention kernel, at most (kMaxGroups + 1 parts of a row block)

// Joins the parts of a row block: o = sum_i w_i O_i / sum_i w_i l_i, w_i = 2^(m_i - max m). blockIdx.x: row block, blockIdx.y: which of gridDim.y
// equal shares of its m_rows * 512 results. The weights of a row are formed first, in one pass over its maxima and sums, so that the loads of the sums
// over the parts do not wait for one another; where a share has fewer pieces of four features than there are threads, several groups of threads take
// every other part and add up in LDS.
__global__ __launch_bounds__(kJoinThreads) void latent_join_kernel(LatentAttnParams p, int m_rows) {
  __shared__ __attribute__((aligned(16))) float sum_o[kJoinThreads][4];
  __shared__ float w_part[2][kMaxGroups + 1], l_part[2][kMaxGroups + 1];
  __shared__ float of_wave[2][kJoinThreads / 64];
  if ((int)blockIdx.x >= *p.items) return;
  const int4 join = p.joins[blockIdx.x];
  if (join.z == join.w) return;
  const int n = join.w / 2 - join.z / 2 + 1;  // parts: slot z, then the even ones up to w
  const auto slot = [&](int i) { return (int64_t)(i == 0 ? join.z : 2 * (join.z / 2 + i)); };
  const int pieces = m_rows * (kLatent / 4) / gridDim.y;  // of this share: a power of two
  const int lanes = min(pieces, kJoinThreads), groups = kJoinThreads / lanes;
  const int mine = threadIdx.x % lanes, group = threadIdx.x / lanes;
  const int n_rows = lanes > kLatent / 4 ? 2 : 1, per_row = kJoinThreads / n_rows;  // rows of a pass, threads that form the weights of each
  const int r = threadIdx.x / per_row, u = threadIdx.x % per_row, waves = per_row / 64;
  for (int piece0 = 0; piece0 < pieces; piece0 += lanes) {
    const int first = blockIdx.y * pieces + piece0;
    const int row = (first + mine) / (kLatent / 4), feature = 4 * ((first + mine) % (kLatent / 4));
    __syncthreads();  // the pass before is through with the shared arrays
    float top = -INFINITY;
    for (int i = u; i < n; i += per_row) {
      const float2 st = p.stats[slot(i) * m_rows + first / (kLatent / 4) + r];
      w_part[r][i] = st.x;
      l_part[r][i] = st.y;
      top = fmaxf(top, st.x);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    of_wave[0][threadIdx.x >> 6] = top;
    __syncthreads();
    for (int k = 0; k < waves; ++k) top = fmaxf(top, of_wave[0][r * waves + k]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int i = u; i < n; i += per_row) {
      const float w = __builtin_amdgcn_exp2f(w_part[r][i] - ref);
      w_part[r][i] = w;
      sum += w * l_part[r][i];
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    of_wave[1][threadIdx.x >> 6] = sum;
    __syncthreads();
    const int rr = n_rows == 2 ? mine / (kLatent / 4) : 0;  // the row of this thread's piece
    sum = 0.f;
    top = -INFINITY;
    for (int k = 0; k < waves; ++k) sum += of_wave[1][rr * waves + k], top = fmaxf(top, of_wave[0][rr * waves + k]);
    f32x4 o = {};
    const float* const src = p.parts + (int64_t)row * kLatent + feature;
    int i = group;
    for (; i + 3 * groups < n; i += 4 * groups) {
      f32x4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const f32x4*>(src + slot(i + k * groups) * m_rows * kLatent);
#pragma unroll
      for (int k = 0; k < 4; ++k) o += x[k] * w_part[rr][i + k * groups];
    }
    for (; i < n; i += groups) o += *reinterpret_cast<const f32x4*>(src + slot(i) * m_rows * kLatent) * w_part[rr][i];
    if (groups > 1) {
      *reinterpret_cast<f32x4*>(sum_o[threadIdx.x]) = o;
      __syncthreads();
      if (group == 0)
        for (int k = 1; k < groups; ++k) o += *reinterpret_cast<const f32x4*>(sum_o[k * lanes + mine]);
    }
    if (group == 0 && row < join.y) {
      const int at = join.x + row, tok = at / p.H, head = at - tok * p.H;
      o = sum == 0.f ? f32x4{} : o * (1.f / sum);
      const u32x2 out = {pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
      *reinterpret_cast<u32x2*>(p.o + (int64_t)tok * p.o_ts + head * p.o_hs + feature) = out;
      if (feature == 0) p.lse[head * p.lse_hs + tok] = sum == 0.f ? -INFINITY : (top == -INFINITY ? 0.f : top) + __builtin_amdgcn_logf(sum);
    }
  }
}

constexpr int kMinTiles = 1;

struct LatentPlan {
  int row_groups;  // of 16 rows a workgroup: 1 or 4
  int groups;      // workgroups of the attention kernel, a multiple of 8
  int max_items;   // row blocks at most
  int join_shares;
  int64_t joins_at, stats_at, parts_at, bytes;  // workspace
};

LatentPlan plan_of(const pith_latent_attn_args* a) {
  LatentPlan pl = {};
  const int64_t rows = a->T * a->H;
  pl.row_groups = rows <= 16 * a->B ? 1 : 4;
  const int m = 16 * pl.row_groups;
  const int64_t items = (rows + m - 1) / m + (a->B < a->T ? a->B : a->T);
  pl.max_items = (int)items;
  const int units = compute_units_or_default() & ~7;
  pl.groups = units < 8 ? 8 : units > kMaxGroups ? kMaxGroups : units;
  int shares = 1;
  while (shares < 4 * m && shares * items < 1024) shares *= 2;
  pl.join_shares = shares;
  const auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  pl.joins_at = 256;
  pl.stats_at = pl.joins_at + up(items * (int64_t)sizeof(int4));
  pl.parts_at = pl.stats_at + up((int64_t)2 * pl.groups * m * sizeof(float2));
  pl.bytes = pl.parts_at + (int64_t)2 * pl.groups * m * kLatent * 4;
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
  const int64_t items = (a->T * a->H + 15) / 16 + a->B;
  if (items * (most / kLatentKeys + 1) > 0x7fffffff - 65536) return fail(PITH_ERR_UNSUPPORTED, "%s: too many row blocks for page tables of that width: call it with fewer tokens at a time", who);
  return PITH_OK;
}

template <int RG>
void launch(const LatentAttnParams& p, bool fp8, bool tree, int groups, hipStream_t s) {
  if (fp8 && tree) latent_attn_kernel<true, true, RG><<<groups, kThreads, 0, s>>>(p);
  else if (fp8) latent_attn_kernel<true, false, RG><<<groups, kThreads, 0, s>>>(p);
  else if (tree) latent_attn_kernel<false, true, RG><<<groups, kThreads, 0, s>>>(p);
  else latent_attn_kernel<false, false, RG><<<groups, kThreads, 0, s>>>(p);
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
  if (pl.row_groups == 1) launch<1>(p, fp8, tree, pl.groups, s);
  else launch<4>(p, fp8, tree, pl.groups, s);
  latent_join_kernel<<<dim3(pl.max_items, pl.join_shares), kJoinThreads, 0, s>>>(p, 16 * pl.row_groups);
  return check_launch(who);
}
