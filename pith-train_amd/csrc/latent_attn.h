// Attention to the latent cache: what its kernels share. The work list, the tiles and the join.
//
// Work list. A sequence of n new tokens and L rows is R = ceil(n H / M) row blocks of M rows (row = token * H + head) times N = ceil(L / K) tiles of K keys,
// and the tiles of all row blocks of all sequences, one behind the other, are dealt to the workgroups in equal ranges. Lengths are read on the device,
// so nothing depends on the host knowing them: a captured call follows its sequences as they grow, and one long sequence among short ones is spread over
// as many workgroups as its share of the tiles.
// To begin and end a row block costs a workgroup the time of several tiles (START: queries, first tile, parts). Where there are fewer row blocks than
// workgroups, ranges can therefore be a little longer and each lie in one row block: every row block is taken for as many tiles as fill whole ranges, LEAST
// tiles or more, the ranges as short as the workgroups allow. The row blocks of a sequence are then cut alike, and as an XCD's workgroups take ranges that
// follow one another, they go through the same tiles at the same time, which its cache fetches about once. Blocks of 64 rows (several a sequence) gain by
// that up to a quarter of their time, so their ranges may be a quarter longer beside the START tiles: a call for 128 heads took 80 us with ranges cut anywhere and
// takes 72, one for trees of up to 48 drafts 192 and 166 (with all tiles in the caches, 67 and 146).
// So how a row's keys are cut follows from the lengths of all sequences of the call, and with that the references, and the order of its sums: the same row in
// another batch may differ in its last bits. Nothing else of one row reaches another: its reference is its own, and so are its infinities and NaN.
// A workgroup whose range covers a row block wholly writes its rows; parts of a row block leave (reference, sum, unnormalised result) in fp32 in the
// workspace, and a second kernel joins them in the order of the keys (results do not depend on scheduling).
#pragma once

#include "attn_tiles.h"
#include "latent_common.h"

namespace pith {

// What the join needs of a row block: its rows (token * H + head of the whole call) and the slots of its parts, the first and, of the workgroups behind
// that one, the last (equal: nothing to join).
struct LatentJoin {
  int row0, rows, first, last;
};

struct LatentAttnParams {
  const __bf16* q_latent;
  const __bf16* q_pe;
  LatentCache cache;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* cu_q;
  const int64_t* tree;
  __bf16* o;
  float* lse;
  int64_t table_rs, q_ts, q_hs, q_pe_ts, q_pe_hs, o_ts, o_hs, lse_hs;
  int T, B, H, table_width;
  int max_len;  // table_width * page_size
  float kappa;  // scale * log2(e)
  // workspace
  int* items;         // number of row blocks of this call
  LatentJoin* joins;  // [row blocks]
  float2* stats;      // [slots][M] reference (in bits) and sum
  float* parts;       // [slots][M * 512] (part_at); slot 2 i: workgroup i's part that begins with its range, 2 i + 1: one that begins later
  int max_items;      // capacity of joins
};

struct SeqWork {
  int tok0, n, len;   // first token, new tokens, cached rows
  int blocks, tiles;  // row blocks, tiles of each
};

// Of tokens c0 .. c1 - 1 and a cached length as the caller gave it.
template <int M, int KEYS>
__device__ __forceinline__ SeqWork seq_work(const LatentAttnParams& p, int c0, int c1, int length) {
  SeqWork s;
  s.tok0 = c0;
  s.n = c1 - c0;
  s.len = min(max(length, 0), p.max_len);
  s.blocks = (s.n * p.H + M - 1) / M;
  s.tiles = max((s.len + KEYS - 1) / KEYS, 1);  // rows without keys get their zeros from an empty tile
  return s;
}
// Token offsets are taken as their maximum so far, so that whatever they hold no token belongs to two sequences, and the work list is no longer than the
// host has made sure of.
__device__ __forceinline__ int token_offset(const LatentAttnParams& p, int i) { return min(max(p.cu_q[i], 0), p.T); }

// Inclusive sums over the lanes of a wavefront.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_dpp(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = add_dpp<0x111, 0xf>(x);  // from 1, 2, 4, 8 lanes below in the row of 16
  x = add_dpp<0x112, 0xf>(x);
  x = add_dpp<0x114, 0xf>(x);
  x = add_dpp<0x118, 0xf>(x);
  x = add_dpp<0x142, 0xa>(x);  // lane 15 of a row to the next row, then lane 31 to the upper half
  return add_dpp<0x143, 0xc>(x);
}

// Inclusive maxima of values from 0 on.
template <int CTRL, int ROWS>
__device__ __forceinline__ int max_dpp(int x) {
  return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_scan_max(int x) {
  x = max_dpp<0x111, 0xf>(x);
  x = max_dpp<0x112, 0xf>(x);
  x = max_dpp<0x114, 0xf>(x);
  x = max_dpp<0x118, 0xf>(x);
  x = max_dpp<0x142, 0xa>(x);
  return max_dpp<0x143, 0xc>(x);
}

// A workgroup's way through its range of the work list, segment by segment (tiles of one row block). Every wave walks for itself; all of it is
// wave-uniform.
template <int M, int KEYS, int START, int LEAST>
struct Walk {
  int range;                // this workgroup's
  int per, begin, at, end;  // length of a range, begin of this one, place, end
  int b, item;              // sequence, row blocks in front of it
  int block, tile;          // row block, first tile of the segment
  bool single;              // one segment a range
  SeqWork s;

  __device__ __forceinline__ int taken(int tiles) const { return single && per > 1 ? (tiles + per - 1) / per * per : tiles; }  // tiles that a row block is taken for

  // False: nothing to do.
  __device__ __forceinline__ bool start(const LatentAttnParams& p, int lane) {
    SeqWork x = {};
    int w = 0, k = 0, sw = 0, sk = 0, total = 0, blocks_total = 0;
    int behind = 0;  // the sequences that were loaded: their last offset
    const auto load = [&](int b0) __attribute__((always_inline)) {  // 64 sequences
      if (b0 == 0) behind = token_offset(p, 0);
      const bool some = b0 + lane < p.B;
      const int c1 = max(wave_scan_max(some ? token_offset(p, b0 + lane + 1) : 0), behind);  // (lanes without one: no tokens)
      x = seq_work<M, KEYS>(p, __builtin_amdgcn_update_dpp(behind, c1, 0x138, 0xf, 0xf, false), c1, some ? p.lengths[b0 + lane] : 0);  // from the lane below
      behind = __builtin_amdgcn_readlane(c1, 63);
    };
    const auto sums = [&]() __attribute__((always_inline)) {
      k = x.blocks;
      w = k * taken(x.tiles);
      sw = wave_scan(w);
      sk = wave_scan(k);
    };
    single = false;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      load(b0);
      sums();
      total += __builtin_amdgcn_readlane(sw, 63);
      blocks_total += __builtin_amdgcn_readlane(sk, 63);
    }
    // (named as global memory: with a store to anywhere behind it, all waits for LDS in the kernel would be waits for everything)
    if (blockIdx.x == 0 && threadIdx.x == 0) *(__attribute__((address_space(1))) int*)(uintptr_t)p.items = min(blocks_total, p.max_items);
    const int groups = gridDim.x;
    range = (blockIdx.x & 7) * (groups >> 3) + (blockIdx.x >> 3);  // an XCD's workgroups (every eighth) take ranges that follow one another
    per = total <= groups ? 1 : __builtin_amdgcn_readfirstlane((total + groups - 1) / groups);  // (divisions leave the scalar registers)
    if (blocks_total < groups && p.B <= 64 && total < 1 << 30) {  // (more sequences are not looked up twice)
      const int most = per + START + (M > 16 ? per / 4 : 0);
      int longer = max(per, LEAST);
      for (int ranges; longer <= most; longer = max(longer + 1, __builtin_amdgcn_readfirstlane((int)(longer * ((float)ranges / groups))))) {
        ranges = __builtin_amdgcn_readlane(wave_scan(k * (longer > 1 ? (x.tiles + longer - 1) / longer : x.tiles)), 63);
        if (ranges <= groups) {
          per = longer;
          single = true;
          if (per > 1) sums();
          break;
        }
      }
    }
    begin = at = range * per;
    end = at + per;  // (the host has bounded total + gridDim.x)
    int before = 0;  // tiles in front of the sequence
    item = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      if (p.B > 64) {
        load(b0);
        sums();
      }
      const uint64_t beyond = __ballot(before + sw > at);
      if (beyond != 0) {
        const int i = __builtin_ctzll(beyond);
        b = b0 + i;
        before += __builtin_amdgcn_readlane(sw - w, i);
        item += __builtin_amdgcn_readlane(sk - k, i);
        s.tok0 = __builtin_amdgcn_readlane(x.tok0, i);
        s.n = __builtin_amdgcn_readlane(x.n, i);
        s.len = __builtin_amdgcn_readlane(x.len, i);
        s.blocks = __builtin_amdgcn_readlane(x.blocks, i);
        s.tiles = __builtin_amdgcn_readlane(x.tiles, i);
        const int each = __builtin_amdgcn_readfirstlane(taken(s.tiles));
        block = __builtin_amdgcn_readfirstlane((at - before) / each);
        tile = at - before - block * each;
        if (!single) end = min(end, total);
        return true;
      }
      before += __builtin_amdgcn_readlane(sw, 63);
      item += __builtin_amdgcn_readlane(sk, 63);
    }
    return false;
  }
  __device__ __forceinline__ int n_tiles() const { return min(s.tiles - tile, end - at); }
  __device__ __forceinline__ int rows(const LatentAttnParams& p) const { return min(s.n * p.H - block * M, M); }
  __device__ __forceinline__ bool whole() const { return n_tiles() == s.tiles; }
  __device__ __forceinline__ int slot() const { return 2 * range + (at == begin ? 0 : 1); }
  // Who ends a row block says how it was cut.
  __device__ __forceinline__ void leave_join(const LatentAttnParams& p) const {
    if (tile + n_tiles() != s.tiles || threadIdx.x != 0 || item + block >= p.max_items) return;
    int first = 0, last = 0;
    if (!whole()) {
      const int from = at - tile;  // of the row block in the work list
      const int id = from / per;
      first = 2 * id + (from == id * per ? 0 : 1);
      last = 2 * range;
    }
    p.joins[item + block] = LatentJoin{s.tok0 * p.H + block * M, rows(p), first, last};
  }
  // On to the next segment. False: the range is done.
  __device__ __forceinline__ bool next(const LatentAttnParams& p) {
    at += n_tiles();
    if (single || at >= end) return false;
    tile = 0;
    if (++block == s.blocks) {
      block = 0;
      item += s.blocks;
      do {
        ++b;
        const int c0 = s.tok0 + s.n;
        s = seq_work<M, KEYS>(p, c0, max(token_offset(p, b + 1), c0), p.lengths[b]);
      } while (s.blocks == 0);
    }
    return true;
  }
};

// ---------------------------------------------------------------------------------------------
// Tiles

template <bool FP8, int KEYS>
struct LatentTile {
  static constexpr int kLatentRow = FP8 ? kLatent : 2 * kLatent;  // bytes
  static constexpr int kPe = KEYS * kLatentRow;                   // offsets in a tile
  static constexpr int kScale = kPe + KEYS * 2 * kRope;           // [KEYS] fp32
  static constexpr int kBytes = kScale + (FP8 ? 256 : 0);         // (tiles begin at multiples of 256)
};

// Latent rows are swizzled by row_swizzle. Rotary rows lie two to a 256-byte LDS row: row 8 w + i and 8 w + 4 + i (i < 4) in pieces 0-7 and 8-15 of LDS
// row 4 w + i, so that eight rows are one instruction; there the fragment reads have no conflict with this swizzle.
__device__ __forceinline__ int pe_row(int row) { return ((row >> 3) << 2) | (row & 3); }
__device__ __forceinline__ int pe_swizzle(int lds_row) { return (lds_row & 3) << 1; }

// Page of the sixteen rows from key on (a multiple of 16), the sequence's last ones where that is behind them. Read as constant memory (nobody writes
// tables while the kernel runs): a scalar load, which the counted waits for tiles do not see.
typedef const __attribute__((address_space(4))) int32_t* ScalarTable;
__device__ __forceinline__ int page_at(const LatentAttnParams& p, ScalarTable table, int key, int last) { return table[min(key, last) >> p.cache.page_shift]; }

// Wave w's (of KEYS / 8) direct loads of a tile: rows 8 w .. 8 w + 7, which are half of the sixteen from key16 = key0 + 16 (w / 2) on; `page`: page_at that.
// Rows behind the sequence's last one come as the page holds them, or the last sixteen again: nobody sees them, and clean_tile takes out what is not finite.
template <bool FP8, int KEYS>
struct TileLoads {
  using T = LatentTile<FP8, KEYS>;
  static constexpr int kLatentLoads = FP8 ? 4 : 8, kLoads = kLatentLoads + (FP8 ? 2 : 1);
  const char *base, *pe;  // of the wave's first row
  const float* scale;
  char* slot;
  int wave;
  __device__ __forceinline__ TileLoads(const LatentAttnParams& p, int page, int key16, int last, char* slot_, int wave_) : slot(slot_), wave(wave_) {
    page = safe_page(__builtin_amdgcn_readfirstlane(page), p.cache.pages);
    const int in_page = (min(key16, last) & ((1 << p.cache.page_shift) - 16)) + 8 * (wave & 1);
    base = p.cache.latent + page * p.cache.latent_ps + (int64_t)in_page * T::kLatentRow;
    pe = reinterpret_cast<const char*>(p.cache.k_pe + page * p.cache.k_pe_ps + (int64_t)in_page * kRope);
    scale = FP8 ? p.cache.scale + page * p.cache.scale_ps + in_page : nullptr;
  }
  // Load n of kLoads, in their order (four latent ones share an M0).
  __device__ __forceinline__ void issue(int n, int lane) const {
    if (n < kLatentLoads) {  // a row, or two of e4m3: 1 KB
      const int r = FP8 ? 2 * n + (lane >> 5) : n;
      const int at = (FP8 ? (lane >> 5) * T::kLatentRow : 0) + (16 * (FP8 ? lane & 31 : lane) ^ 16 * row_swizzle(8 * wave + r));
      const char* const four = base + (n & ~3) * 1024;
      if ((n & 3) == 0) load_lds16(four, at, slot + 8 * wave * T::kLatentRow + n * 1024);
      else if ((n & 3) == 1) load_lds16_next<1024>(four, at);
      else if ((n & 3) == 2) load_lds16_next<2 * 1024>(four, at);
      else load_lds16_next<3 * 1024>(four, at);
    } else if (n == kLatentLoads) {
      const int piece = (lane & 15) ^ pe_swizzle(4 * wave + (lane >> 4));
      load_lds16(pe, (4 * (piece >> 3) + (lane >> 4)) * (2 * kRope) + 16 * (piece & 7), slot + T::kPe + wave * 1024);
    } else {
      if (lane < 8) load_lds4(scale + lane, slot + T::kScale + 32 * wave);
    }
  }
  __device__ __forceinline__ void issue_all(int lane) const {
    asm volatile("" : "+v"(lane));  // the rows' offsets are formed on the spot, not kept (and spilled) from tile to tile
#pragma unroll
    for (int n = 0; n < kLoads; ++n) issue(n, lane);
  }
};

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

// Eight e4m3 values (two words) -> bf16, exact.
__device__ __forceinline__ bf16x8 widen(uint32_t w0, uint32_t w1) {
  const bf16x2 a = fp8x2_to_bf16<false>(w0), b = fp8x2_to_bf16<true>(w0), c = fp8x2_to_bf16<false>(w1), d = fp8x2_to_bf16<true>(w1);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A wave's products of values: product n's result v in a lane of group g is feature 16 n + 4 g + v of its 128. (Dealt so that a lane's results of two
// products are eight consecutive features, the transposed bf16 reads take halves of four pieces of a row and conflict in the banks.)
// Place of the lane's transposed reads of 128 features in a tile, rows 0-31, wave w's from feature 128 w on; those of other products and rows are
// ^ and + from there. A read brings four columns (bf16) or eight (e4m3) of a row.
template <bool FP8>
__device__ __forceinline__ int value_place(int wave, int c, int g) {
  const int r = 8 * g + (FP8 ? c >> 1 : c >> 2);
  const int piece = FP8 ? 8 * wave : 16 * wave + ((c >> 1) & 1);
  return r * (FP8 ? kLatent : 2 * kLatent) + ((piece ^ row_swizzle(r)) << 4) + 8 * (c & 1);
}

// Operand A of product n over keys 8 g + e; `first`: lds_address of the tile + value_place.
template <bool FP8>
__device__ __forceinline__ bf16x8 value_fragment(uint32_t first, int n) {
  if constexpr (FP8) {
    typedef __attribute__((ext_vector_type(2))) int i32x2;
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(uintptr_t)(first ^ (16 * n)));
    return widen((uint32_t)raw[0], (uint32_t)raw[1]);
  } else {  // four rows further on the swizzle differs in its highest bit
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(first ^ (32 * n)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((first ^ (32 * n ^ 128)) + 4 * (2 * kLatent)));
    typedef __attribute__((ext_vector_type(8))) short s16x8;
    return __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }
}

// Infinities and NaN of a wave's 128 features from 128 w on, in all 32 rows of a tile -> 0, in place. For tiles that some rows see in part only: a row's weight
// of a key it does not see is 0, and must stay so against whatever the key holds. A row that sees such a key has a score of the same kind.
template <bool FP8>
__device__ __forceinline__ void clean_tile(char* tile, int w, int lane) {
  constexpr int kPieces = FP8 ? 8 : 16;  // of a row
#pragma unroll 1
  for (int i0 = lane; i0 < 32 * kPieces; i0 += 4 * 64) {  // four a lane at a time
    u32x4 x[4];
    char* at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + 64 * j, row = i / kPieces, piece = kPieces * w + i % kPieces;
      at[j] = tile + row * LatentTile<FP8, 32>::kLatentRow + ((piece ^ row_swizzle(row)) << 4);
      x[j] = *reinterpret_cast<const u32x4*>(at[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (FP8) {
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (((x[j][e] >> k) & 0x7fu) == 0x7fu) x[j][e] &= ~(0xffu << k);
        } else {
          if ((x[j][e] & 0x7f80u) == 0x7f80u) x[j][e] &= 0xffff0000u;
          if ((x[j][e] & 0x7f800000u) == 0x7f800000u) x[j][e] &= 0xffffu;
        }
      }
      *reinterpret_cast<u32x4*>(at[j]) = x[j];
    }
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

// Scores x[0 .. N-1] of keys key0 .. against a row of token tok: those of keys that it does not see -> -infinity. In the last tiles of a sequence only, so
// what a token sees is looked up anew there. (In words and without branches: hipcc 7.2 lost the selected score behind nested conditions on a shift of
// 64 bits.)
template <bool TREE, int N, typename X>
__device__ __forceinline__ void mask_scores(const LatentAttnParams& p, const SeqWork& s, X& x, int tok, int key0) {
  uint32_t lo = 0, hi = 0;
  if constexpr (TREE) {
    const uint64_t word = (uint64_t)p.tree[s.tok0 + tok];
    lo = (uint32_t)word;
    hi = (uint32_t)(word >> 32);
  }
  const int ctx = s.len - s.n;  // rows in front of the new ones (below zero only where the lengths contradict each other)
#pragma unroll
  for (int v = 0; v < N; ++v) {
    const int key = key0 + v, draft = key - ctx;
    int seen;
    if constexpr (TREE) {
      const uint32_t bits = draft < 32 ? lo : hi;
      seen = (draft < 0) | ((draft < 64) & (int)((bits >> (draft & 31)) & 1u));
    } else {
      seen = draft <= tok;
    }
    seen &= key < s.len;
    x[v] = seen ? x[v] : -INFINITY;
  }
}

// Whether some row may not see all of the tile from key0 on.
template <bool TREE, int KEYS>
__device__ __forceinline__ bool partial_tile(const SeqWork& s, int key0) { return key0 + KEYS > s.len - s.n + (TREE ? 0 : 1); }

// The lane's number, formed on the spot: it (and what follows from it) takes no register from tile to tile.
__device__ __forceinline__ int lane_here() {
  int lane;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  return lane;
}

// A wave-uniform address that the compiler formed in vector registers.
__device__ __forceinline__ const char* scalar_pointer(const void* x) {
  const uint64_t a = reinterpret_cast<uint64_t>(x);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return reinterpret_cast<const char*>((uint64_t)hi << 32 | lo);
}

// Query rows row0 .. of the walk's row block into LDS, laid out like the rows of a bf16 tile of M keys: wave w brings rows 8 w .. 8 w + 7 (M = 16: the first
// two waves). Fetched straight into registers, a fragment touches 16 rows, every lane of a quad on a line of its own, which the address unit serves
// at one lane a cycle: the 36 fragments of 64 rows took a workgroup 9 us in front of its first tile. Rows behind the block's last one are that one.
template <int M, typename W>
__device__ __forceinline__ void stage_queries(const LatentAttnParams& p, const W& walk, char* area, int wave, int lane) {
  using T = LatentTile<false, M>;
  if (8 * wave >= M) return;
  const int last = walk.rows(p) - 1, row0 = walk.block * M;
  int tok = __builtin_amdgcn_readfirstlane((row0 + min(8 * wave, last)) / p.H), head = row0 + min(8 * wave, last) - tok * p.H;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    load_lds16(scalar_pointer(p.q_latent + (int64_t)(walk.s.tok0 + tok) * p.q_ts + head * p.q_hs), (16 * lane) ^ (16 * row_swizzle(8 * wave + i)),
               area + (8 * wave + i) * T::kLatentRow);
    if (8 * wave + i < last && ++head == p.H) head = 0, ++tok;
  }
  const int piece = (lane & 15) ^ pe_swizzle(4 * wave + (lane >> 4));
  const int row = row0 + min(8 * wave + 4 * (piece >> 3) + (lane >> 4), last);
  const int t = row / p.H, h = row - t * p.H;
  load_lds16_at(p.q_pe + (int64_t)(walk.s.tok0 + t) * p.q_pe_ts + h * p.q_pe_hs + 8 * (piece & 7), area + T::kPe + wave * 1024);
}

// Operand B fragments of staged row `row`: 32 latent features a step from `latent` on (e4m3 keys are read 16 features at a time: steps 2 i, 2 i + 1 then
// contract features 64 i + 16 g + {0..7, 8..15}), then two rotary steps.
template <bool FP8, int M, int Q>
__device__ __forceinline__ void read_query(const char* area, int row, int latent, int g, bf16x8 (&q)[Q]) {
  using T = LatentTile<false, M>;
  asm volatile("" : "+v"(row), "+v"(g));  // the places are formed here, not kept (and spilled) from segment to segment
  const char* const rows = area + row * T::kLatentRow + 2 * latent;
#pragma unroll
  for (int i = 0; i < Q - 2; ++i) {
    const int piece = FP8 ? 8 * (i >> 1) + 2 * g + (i & 1) : 4 * i + g;
    q[i] = *reinterpret_cast<const bf16x8*>(rows + ((piece ^ row_swizzle(row)) << 4));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    q[Q - 2 + i] = *reinterpret_cast<const bf16x8*>(area + T::kPe + pe_row(row) * 256 + (((8 * ((row >> 2) & 1) + 4 * i + g) ^ pe_swizzle(pe_row(row))) << 4));
}

// Results of a lane's row of group r (the wave's 128 features) as bf16, and its lse by one lane; or, where the segment is a part, reference, sum and
// unnormalised results in the workspace: there result vector n of a wave (features 16 (8 wave + n) ..) lies as the wave holds it, 16 bytes a lane
// (part_at), because row by row an instruction would touch 16 of them.
template <int M>
__device__ __forceinline__ int64_t part_at(int64_t slot, int group, int vector, int lane) {  // vector: 8 wave + n; in floats
  return ((slot * (M / 16) + group) * (kLatent / 16) + vector) * 256 + 4 * lane;
}
template <int M, typename W>
__device__ __forceinline__ void store_row(const LatentAttnParams& p, const W& walk, const f32x4 (&acc)[8], float top, float sum, int r, int wave, int lane) {
  const int row = 16 * r + (lane & 15), g = lane >> 4;
  const bool first = wave == 0 && g == 0;
  if (walk.whole()) {
    if (row >= walk.rows(p)) return;
    const int at = walk.block * M + row, tok = walk.s.tok0 + at / p.H, head = at % p.H;
    const float inv = 1.f / sum;
    __bf16* const dst = p.o + (int64_t)tok * p.o_ts + head * p.o_hs + 128 * wave + 4 * g;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const f32x4 x = sum == 0.f ? f32x4{} : acc[n] * inv;
      *reinterpret_cast<u32x2*>(dst + 16 * n) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
    }
    if (first) p.lse[head * p.lse_hs + tok] = sum == 0.f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
  } else {
    const int64_t slot = walk.slot();
#pragma unroll
    for (int n = 0; n < 8; ++n) *reinterpret_cast<f32x4*>(p.parts + part_at<M>(slot, r, 8 * wave + n, lane)) = acc[n];
    if (first) p.stats[slot * M + row] = make_float2(top, sum);
  }
}

// Where a score may exceed the reference of its row's weights, in bits, before the reference is moved: weights stay below 2^8, far from the end of
// their range, and neither they nor the sums lose precision by it.
constexpr float kSlack = 8.f;
// A row's reference behind scores of up to `top`; it stands unless they are beyond the slack, whatever other rows do (no row's result depends on another's).
__device__ __forceinline__ float moved(float reference, float top) { return top > reference + kSlack ? top : reference; }

// The attention kernel for 64 rows to a workgroup (latent_attn_wide.hip).
constexpr int kWideRows = 64;
void launch_latent_wide(const LatentAttnParams& p, bool fp8, bool tree, int groups, hipStream_t stream);

}  // namespace pith
