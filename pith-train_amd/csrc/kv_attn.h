// Attention of new tokens to the rows of a key-value cache: the work list, the kernel, and what its join needs.
//
//   S = kappa Q K^T,  O = softmax(S) V        for the query heads that share a key-value head
//
// Work list. The query rows of a sequence and key-value head (row = token * group + head of the group, n tokens: n * group rows) are cut into row blocks of
// M = 16, 32 or 64 rows, each of which goes through the sequence's keys in steps of 128; the steps of all row blocks, one behind the other, are dealt
// to the workgroups in equal ranges. Lengths are read on the device, so nothing depends on the host knowing them: a captured call follows its sequences as
// they grow, and one long sequence among short ones is spread over as many workgroups as its share of the steps. Where there are fewer row blocks than
// workgroups, ranges may be a little longer and each lie in one row block (to begin one costs queries, a first tile and a part). An XCD's workgroups take
// ranges that follow one another, so that row blocks of one head find each other's keys in its cache.
// Steps that no row of a block sees (of a prompt's first tokens, behind them) are dealt like the others but not taken; the row blocks' order puts the first and the
// last beside each other, so that ranges of two or more are as much work all the same (4 prompts of 2048 tokens, heads of 32 / 4: 782 us without either, 476 with, when both came).
// Two kinds of calls need no such list. Where page tables are so short that no row block is worth cutting, every workgroup takes one, whole, and there is
// nothing to join. And tables of the heads (selected pages) are nearly full for whoever has a long context, so their row blocks are cut into the same
// number of parts each, as many as there are workgroups for.
// A workgroup whose range covers a row block wholly writes its rows; parts leave (reference, sum, unnormalised result) in fp32 in the workspace, and a second
// kernel joins them in the order of the keys (results do not depend on scheduling). So how a row's keys are cut, its references and the order of its sums
// follow from the lengths of all sequences of the call; nothing else of one row reaches another.
//
// The kernel. Memory bounds it: a key row and a value row of 512 bytes (bf16, 128 features) stand against 4 * 128 flop for each of the group's rows. So the four
// wavefronts of a workgroup walk alone, each through every fourth tile of 32 keys, with no barrier until the segment ends: a wave brings its tiles global -> LDS by
// direct loads into a ring of its own (see KVRing) and waits with counted waits for its own requests only, for the keys while the values are
// still under way. Products are 16x16x32 with the query row as the result's column, so a lane owns one row, and the scores of a lane are
// its part of operand B of the second product as they stand: key 4 g + v of either half tile is contracted at place 8 g + v or 8 g + 4 + v, and the values are read
// (transposed, from LDS) in that order. No weight moves between lanes. The waves' results of a segment are joined through LDS.
// A fragment that was read serves all 16-row groups of the block: 64 rows cost a tile's reads once. With M = 64 the products are 1024 of a tile's cycles, and
// the tile still comes more slowly than that from memory.
// Measured, heads of 32 / 4 with 128 features: 32 sequences of up to 8192 rows, bf16, one token each (303 MB) 64 us, 4.7 TB/s; 8 of up to 131072 rows, e4m3 (879 MB)
// 160 us, 5.5 TB/s, where a copy reaches 4.9; 64 selected pages of 8 such sequences (34 MB) 15 us, of which the join's launch is 4 and beginnings and ends
// about 4; one sequence of 517 rows 9.7 us, a launch and 5 steps, each of which waits for memory.
// The matrix cores take weights as bf16 beside a cache of bf16 (or e4m3, widened exactly; a weight then has its row's scale in it). In blocks of 16 rows, where these
// products are few beside the bytes, a weight goes in as two numbers, its upper half and the rest rounded, and keeps 16 bits of its fraction: 2^-15 of it is lost at
// most, and the outputs are off by what their own rounding does (norm of the difference from 64 bits by the norm: 0.0016; 0.0023 with one number). It takes, us with one
// number / two: one sequence of 517 rows 8.9 / 9.7 (eight more products and 20 instructions a tile in a chain of five), 32 of up to 8192 63.0 / 63.5, 8 of up to
// 131072, e4m3, 158.2 / 158.8, 1024 of up to 200 73.1 / 74.9, 64 selected pages 15.2 / 15.2. Blocks of 32 and 64 rows take one number, half a step, 2^-8, of each: there the
// second costs 2 to 19 % (8 tokens, 32 x 8192 rows 111.5 / 114.1, 16, 16 x 8192, e4m3, 78.9 / 84.7, 512 behind 8192 111 / 133, 4 prompts of 2048 227 / 255, half of them cached).
// The sum of the weights is of the unrounded ones everywhere.
#pragma once

#include "cache_attn.h"
#include "kv_common.h"

#include <type_traits>

namespace pith {

constexpr int kKVThreads = 256, kKVWaves = 4;
constexpr int kTileKeys = 32, kStepKeys = kKVWaves * kTileKeys;

// What the join needs of a row block: first of its rows within the sequence and head, first token and head of that, its rows, and its parts: the slot of the
// first, that of the second, and the slots from one to the next (parts = 1: nothing to join).
struct KVJoin {
  int row0, tok0, head, rows, first, second, stride, parts;
};

struct KVAttnParams {
  const __bf16* q;
  KVCache cache;
  const int32_t *table, *lengths, *cu_q;
  const int64_t* tree;
  __bf16* o;
  float* lse;
  int64_t table_rs, table_hs, q_ts, q_hs, o_ts, o_hs, lse_hs;
  int T, B, H, group, table_width;
  int head_tables;  // key-value heads with tables of their own, or 1: tables of all
  int max_len;      // table_width * page_size
  float kappa;      // scale * log2(e)
  int whole;        // steps of the longest row block where none is cut, else 0
  int parts;        // of every row block, where all are cut alike (into two or more), else 0
  // workspace (not used where none is cut)
  int* items;        // number of entries of joins in this call
  KVJoin* joins;     // one for every row block, or, where those may be more, for every workgroup that its range's first segment (no other can end a row block that is cut)
  float2* stats;     // [slots][M] reference (in bits) and sum
  float* results;    // [slots][M][D] of parts; slot 2 i: of workgroup i's that begins with its range, 2 i + 1: one that begins later (cut alike: slot i)
  int max_items;     // capacity of joins
  int by_range;      // joins are the workgroups'
};

// A sequence, or a sequence's key-value head where these have tables of their own.
struct KVWork {
  int tok0, n, len;   // first token, new tokens, cached rows
  int blocks, steps;  // row blocks of all its heads, steps of each
};

template <int M>
__device__ __forceinline__ KVWork kv_work(const KVAttnParams& p, int c0, int c1, int length) {
  KVWork s;
  s.tok0 = c0;
  s.n = c1 - c0;
  s.len = min(max(length, 0), p.max_len);
  s.blocks = (s.n * p.group + M - 1) / M * (p.head_tables > 1 ? 1 : p.cache.heads);
  s.steps = max((s.len + kStepKeys - 1) / kStepKeys, 1);  // rows without keys get their zeros from an empty step
  return s;
}
// Token offsets are taken as their maximum so far, so that whatever they hold no token belongs to two sequences, and the work list is no longer than the
// host has made sure of.
__device__ __forceinline__ int kv_offset(const KVAttnParams& p, int b) { return p.cu_q ? min(max(p.cu_q[b], 0), p.T) : b; }

// A workgroup's way through its range of the work list, segment by segment (steps of one row block). Every wave walks for itself; all of it is wave-uniform.
template <int M>
struct KVWalk {
  static constexpr int kStart = 2;  // steps that a range may be longer
  int range, per, begin, at, end;  // this workgroup's range, its length, begin, place, end
  int seq, item, block, step;      // sequence, row blocks in front of it, row block, first step of the segment
  bool single;                     // one segment a range
  KVWork s;

  __device__ __forceinline__ int taken(int steps) const { return single && per > 1 ? (steps + per - 1) / per * per : steps; }  // steps that a row block is taken for

  // False: nothing to do.
  __device__ __forceinline__ bool start(const KVAttnParams& p, int lane) {
    const int groups = gridDim.x;
    range = (blockIdx.x & 7) * (groups >> 3) + (blockIdx.x >> 3);  // an XCD's workgroups (every eighth) take ranges that follow one another
    const auto uniform = [](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(v); };
    if (!p.cu_q && (p.whole || p.parts)) {  // one token a sequence: all have the same number of row blocks
      const int parts = p.parts ? p.parts : 1, each = (p.group + M - 1) / M * (p.head_tables > 1 ? 1 : p.cache.heads);
      const int all = uniform(range / parts), part = range - all * parts;
      seq = uniform(all / each);
      if (seq >= p.B * p.head_tables) return false;
      block = all - seq * each;
      item = seq * each;
      const int b = uniform(p.head_tables > 1 ? seq / p.head_tables : seq);
      s = kv_work<M>(p, b, b + 1, uniform(p.lengths[seq]));
      per = uniform((s.steps + parts - 1) / parts);
      step = begin = at = part * per;  // (beyond the row block's last step: a part without keys)
      end = at + per;
      single = true;
      if (p.parts && blockIdx.x == 0 && threadIdx.x == 0) *(__attribute__((address_space(1))) int*)(uintptr_t)p.items = min(p.B * p.head_tables * each, p.max_items);
      return true;
    }
    KVWork x = {};
    int w = 0, k = 0, sw = 0, sk = 0, total = 0, blocks_total = 0;
    int behind = kv_offset(p, 0);  // the sequences that were digested: their last offset
    const auto fetch = [&](int b0, int& length, int& end) __attribute__((always_inline)) {  // of 64 sequences
      const int b = min(b0 + lane, p.B - 1);
      length = p.lengths[b];
      end = kv_offset(p, b + 1);
    };
    const auto digest = [&](int b0, int length, int end) __attribute__((always_inline)) {
      const bool some = b0 + lane < p.B;
      const int c1 = max(wave_scan_max(some ? end : 0), behind);  // (lanes without one: no tokens)
      x = kv_work<M>(p, __builtin_amdgcn_update_dpp(behind, c1, 0x138, 0xf, 0xf, false), c1, some ? length : 0);  // from the lane below
      behind = __builtin_amdgcn_readlane(c1, 63);
    };
    const auto sums = [&]() __attribute__((always_inline)) {
      k = x.blocks;
      w = k * taken(x.steps);
      sw = wave_scan(w);
      sk = wave_scan(k);
    };
    single = p.whole != 0;
    per = p.whole;
    // Lane i: steps, row blocks and last offset of the first i + 1 times 64 sequences (of the first 4096).
    int steps_to = 0, blocks_to = 0, offset_to = 0;
    const auto add = [&]() __attribute__((always_inline)) {
      sums();
      total += __builtin_amdgcn_readlane(sw, 63);
      blocks_total += __builtin_amdgcn_readlane(sk, 63);
    };
    if (p.B <= 64) {
      int length, end;
      fetch(0, length, end);
      digest(0, length, end);
      add();
    } else {
#pragma unroll 1
      for (int b0 = 0; b0 < p.B; b0 += 256) {
        int length[4], end[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) fetch(b0 + 64 * j, length[j], end[j]);  // (four loads at a time: those behind the last sequence are its own)
#pragma unroll 1
        for (int j = 0; j < 4 && b0 + 64 * j < p.B; ++j) {
          digest(b0 + 64 * j, length[0], end[0]);
          add();
          const bool mine = lane == (b0 >> 6) + j;
          steps_to = mine ? total : steps_to, blocks_to = mine ? blocks_total : blocks_to, offset_to = mine ? behind : offset_to;
          length[0] = length[1], length[1] = length[2], length[2] = length[3];
          end[0] = end[1], end[1] = end[2], end[2] = end[3];
        }
      }
    }
    if (!p.whole) {
      per = total <= groups ? 1 : uniform((total + groups - 1) / groups);  // (divisions leave the scalar registers)
      if (blocks_total < groups && p.B <= 64 && total < 1 << 30) {  // (more sequences are not looked up twice)
        const int most = per + kStart;
        int longer = per;
#pragma unroll 1
        for (int ranges; longer <= most; longer = max(longer + 1, uniform((int)(longer * ((float)ranges / groups))))) {
          ranges = __builtin_amdgcn_readlane(wave_scan(k * (longer > 1 ? (x.steps + longer - 1) / longer : x.steps)), 63);
          if (ranges <= groups) {
            per = longer;
            single = true;
            if (per > 1) sums();
            total = ranges * per;  // with what row blocks are taken for
            break;
          }
        }
      }
      // (named as global memory: with a store to anywhere behind it, all waits for LDS in the kernel would be waits for everything)
      if (blockIdx.x == 0 && threadIdx.x == 0)
        *(__attribute__((address_space(1))) int*)(uintptr_t)p.items = min(p.by_range ? uniform((total + per - 1) / per) : blocks_total, p.max_items);
    }
    begin = at = range * per;
    end = at + per;  // (the host has bounded total + gridDim.x)
    int before = 0, b0 = 0;  // steps in front of the sequence; the first of the 64 that it may be among
    item = 0;
    if (p.B > 64) {
      const int chunks = min(__popcll(__ballot(steps_to <= at && 64 * lane < p.B)), 63);  // (steps only grow; lanes without sequences are behind)
      if (chunks > 0) {
        before = __builtin_amdgcn_readlane(steps_to, chunks - 1);
        item = __builtin_amdgcn_readlane(blocks_to, chunks - 1);
        behind = __builtin_amdgcn_readlane(offset_to, chunks - 1);
        b0 = 64 * chunks;
      } else {
        behind = kv_offset(p, 0);
      }
    }
#pragma unroll 1
    for (; b0 < p.B; b0 += 64) {
      if (p.B > 64) {
        int length, end;
        fetch(b0, length, end);
        digest(b0, length, end);
        sums();
      }
      const uint64_t beyond = __ballot(before + sw > at);
      if (beyond != 0) {
        const int i = __builtin_ctzll(beyond);
        seq = b0 + i;
        before += __builtin_amdgcn_readlane(sw - w, i);
        item += __builtin_amdgcn_readlane(sk - k, i);
        s.tok0 = __builtin_amdgcn_readlane(x.tok0, i);
        s.n = __builtin_amdgcn_readlane(x.n, i);
        s.len = __builtin_amdgcn_readlane(x.len, i);
        s.blocks = __builtin_amdgcn_readlane(x.blocks, i);
        s.steps = __builtin_amdgcn_readlane(x.steps, i);
        const int each = uniform(taken(s.steps));
        block = uniform((at - before) / each);
        step = at - before - block * each;
        if (!single) end = min(end, total);
        return true;
      }
      before += __builtin_amdgcn_readlane(sw, 63);
      item += __builtin_amdgcn_readlane(sk, 63);
    }
    return false;
  }
  __device__ __forceinline__ int n_steps() const { return min(s.steps - step, end - at); }  // (a part without keys: 0 or less)
  __device__ __forceinline__ bool whole(const KVAttnParams& p) const { return !p.parts && n_steps() == s.steps; }
  __device__ __forceinline__ int slot(const KVAttnParams& p) const { return p.parts ? range : 2 * range + (at == begin ? 0 : 1); }
  // Who ends a row block says how it was cut; by ranges, everybody says once whether it has ended one.
  __device__ __forceinline__ void leave_join(const KVAttnParams& p, int row0, int head, int rows) const {
    const int index = p.by_range ? range : item + block;
    if (p.whole || threadIdx.x != 0 || index >= p.max_items || (p.by_range && at != begin)) return;
    KVJoin join = {row0, s.tok0, head, rows, 0, 0, 0, 1};
    if (p.parts) {
      if (step != 0) return;
      join.first = range, join.second = range + 1, join.stride = 1, join.parts = p.parts;
    } else if (step + n_steps() == s.steps) {
      if (!whole(p)) {
        const int from = at - step;  // of the row block in the work list
        const int id = from / per;
        join.first = 2 * id + (from == id * per ? 0 : 1);
        join.second = 2 * id + 2, join.stride = 2, join.parts = range - id + 1;
      }
    } else if (!p.by_range) {
      return;
    }
    p.joins[index] = join;
  }
  // On to the next segment. False: the range is done.
  __device__ __forceinline__ bool next(const KVAttnParams& p) {
    at += n_steps();
    if (single || at >= end) return false;
    step = 0;
    if (++block == s.blocks) {
      block = 0;
      item += s.blocks;
      do {
        ++seq;
        const int c0 = s.tok0 + s.n;
        s = kv_work<M>(p, c0, max(kv_offset(p, seq + 1), c0), p.lengths[seq]);
      } while (s.blocks == 0);
    }
    return true;
  }
};

// ---------------------------------------------------------------------------------------------
// Tiles

// 32 rows of keys or of values, packed: rows of 256, 128 or 64 bytes lie 1, 2 or 4 to an LDS line of 256. Piece (16 bytes) q of row r lies at q ^ swizzle(r) of
// its row. LDS serves 256 bytes a cycle, and a wavefront's 16-byte reads as lanes 0-3 12-15 20-27, then 4-11 16-19 28-31, and the upper half alike, 8-byte
// reads by halves. The fragment reads of keys (lane c + 16 g: row c, piece q + g) then have rows {0-3, 12-15} at piece q and {4-11} at q + 1, and the
// transposed reads of values rows 0-7 (bf16; two pieces each) or 0-7 and 16-23 (e4m3; one piece each): no two on one bank in either.
template <int ROW>
__device__ __forceinline__ constexpr int kv_swizzle(int r) {
  return ROW == 256 ? 2 * (r & 7) : ROW == 128 ? 2 * ((r >> 1) & 3) | ((r >> 4) & 1) : 2 * ((r >> 2) & 1) | ((r >> 4) & 1);
}

template <int D, bool FP8>
struct KVTile {
  static constexpr int kRow = FP8 ? D : 2 * D;                // bytes
  static constexpr int kBytes = kTileKeys * kRow;             // of keys, and of values
  static constexpr int kLoads = kBytes / 1024;                // instructions of a wave, for either
  static constexpr int kScaleLoads = FP8 ? 1 : 0;             // 32 scales of keys and 32 of values
  static constexpr int kScaleBytes = FP8 ? 256 : 0;
  static constexpr int kSlot = 2 * kBytes + kScaleBytes;
  static constexpr int kAll = kScaleLoads + 2 * kLoads;       // requests of a tile

  // Place in the source, within 16 rows, of what lane `lane` brings in instruction 0; that of instruction n is ^ (source_xor(n)) and 1024 n behind.
  static __device__ __forceinline__ int source(int lane) {
    constexpr int kPieces = kRow / 16, kRows = 256 / kRow;  // of a row, of a line
    const int row = kRows * (lane >> 4) + (lane & 15) / kPieces, piece = (lane & 15) % kPieces;
    return row * kRow + ((piece ^ kv_swizzle<kRow>(row)) << 4);
  }
  static __device__ __forceinline__ constexpr int source_xor(int n) { return kRow == 256 ? 128 * (n & 1) : kRow == 128 ? 16 * (n >> 1) : 16 * n; }
  // Place in a tile of piece q of row r (< 32).
  static __device__ __forceinline__ int place(int r, int q) { return r * kRow + ((q ^ kv_swizzle<kRow>(r)) << 4); }
};

// Tiles of a wave in flight, and workgroups of a compute unit. Two workgroups fill each other's gaps (their beginnings and ends, a wave's way from its keys to its
// weights), and a ring of one tile is enough then, as its keys are asked for while the values before them are worked on and the other way round. 64 rows fill the
// registers, and with them one workgroup has the compute unit, with rings of 128 KB. (us with one workgroup
// and rings of 128 KB / with two and 64 KB each / with two and one tile a wave: 8 sequences of 64 selected pages, e4m3, 17.2 / 15.3 / 15.2; trees of 8 over 5001 rows, heads
// of 64, 16.8 / 15.9 / 15.6; 4 tokens, 32 x 1024 rows 23.2 / 18.6; 8 x 131072 rows, e4m3, 165 / 164 / 160, heads of 64 - / 95 / 88; 1 x 9094 - / 14.2 / 15.1. Three or four
// workgroups, where their registers allow: 16.8 for the trees, 165 for the long rows.)
template <int D, bool FP8, int R>
struct KVRing {
  static constexpr int kPerUnit = R <= 2 ? 2 : 1;
  static constexpr int kSlots = R > 2 ? 2 : 1;
  static constexpr int kBytes = kSlots * KVTile<D, FP8>::kSlot;
};

// A wave's requests for the 32 rows from key on (a multiple of 32): two times sixteen rows, each of one page. Rows behind the sequence's last one come as the
// page holds them, or the last sixteen again: nobody sees them, and clean_values takes out what is not finite.
template <int D, bool FP8>
struct KVLoads {
  using T = KVTile<D, FP8>;
  int64_t page[2];
  int in_page[2];
  __device__ __forceinline__ KVLoads(const KVAttnParams& p, const int (&page_)[2], int key, int last, int head) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      page[h] = safe_page(__builtin_amdgcn_readfirstlane(page_[h]), p.cache.pages);
      in_page[h] = (head << p.cache.page_shift) + (min(key + 16 * h, last) & ((1 << p.cache.page_shift) - 16));
    }
  }
  __device__ __forceinline__ void rows(const char* base, int64_t page_bytes, char* dst, int source) const {
#pragma unroll
    for (int n = 0; n < T::kLoads; ++n) {
      constexpr int kPerHalf = T::kLoads / 2;
      const int h = n / kPerHalf, i = n % kPerHalf;
      const char* const from = base + page[h] * page_bytes + (int64_t)in_page[h] * T::kRow;
      const int at = source ^ T::source_xor(n);
      if (i == 0) load_lds16(from, at, dst + n * 1024);
      else if (i == 1) load_lds16_next<1024>(from, at);
      else if (i == 2) load_lds16_next<2 * 1024>(from, at);
      else load_lds16_next<3 * 1024>(from, at);
    }
  }
  __device__ __forceinline__ void keys(const KVAttnParams& p, char* slot, int source, int lane) const {
    if constexpr (FP8) {  // scales: lanes 0-31 of the keys, 32-63 of the values
      const int h = (lane >> 4) & 1;
      const float* const from = lane < 32 ? p.cache.k_scale + (h ? page[1] * p.cache.k_scale_ps + in_page[1] : page[0] * p.cache.k_scale_ps + in_page[0])
                                          : p.cache.v_scale + (h ? page[1] * p.cache.v_scale_ps + in_page[1] : page[0] * p.cache.v_scale_ps + in_page[0]);
      load_lds4(from + (lane & 15), slot + 2 * T::kBytes);
    }
    rows(p.cache.k, p.cache.k_ps, slot, source);
  }
  __device__ __forceinline__ void values(const KVAttnParams& p, char* slot, int source) const { rows(p.cache.v, p.cache.v_ps, slot + T::kBytes, source); }
};

// Query rows row0 .. of a sequence and head into LDS, laid out like keys of bf16: 1 KB a request, every lane from an address of its own, the waves in turn. (Loads of the
// compiler's would make it wait for everything that is under way at their first use, in every turn of the loop.) Rows behind the block's last one are that one.
template <int D, int R>
struct KVQueries {
  static constexpr int kBytes = 16 * R * 2 * D, kAll = kBytes / 1024, kEach = kAll > kKVWaves ? kAll / kKVWaves : 1;  // requests; of a wave (fewer than waves: some twice)
  static __device__ __forceinline__ void stage(const KVAttnParams& p, const KVWork& s, int head, int row0, int rows, char* area, int wave, int lane) {
    using T = KVTile<D, false>;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int n = (wave * kEach + j) % kAll;
      const int row = (1024 * n + 16 * lane) / T::kRow, piece = (lane % (T::kRow / 16)) ^ (kv_swizzle<T::kRow>(row));
      const int at = row0 + min(row, rows - 1), tok = at / p.group;
      load_lds16_at(p.q + (int64_t)(s.tok0 + tok) * p.q_ts + (int64_t)(head * p.group + at - tok * p.group) * p.q_hs + 8 * piece, area + 1024 * n);
    }
  }
};

// Until all but the last `later` tiles' requests and EXTRA more are there.
template <int D, bool FP8, int SLOTS, int EXTRA>
__device__ __forceinline__ void wait_tiles(int later) {
  static_assert(SLOTS <= 2, "at most one tile behind");
  if (SLOTS == 2 && later >= 1) wait_loads<KVTile<D, FP8>::kAll + EXTRA>();
  else wait_loads<EXTRA>();
}

// Operand A over 32 keys, features 16 n ..; `first`: lds_address of the values + the lane's place. Element 4 h + v: key 16 h + 4 g + v.
template <int D, bool FP8>
__device__ __forceinline__ int kv_value_place(int c, int g) {
  if constexpr (FP8) {
    const int r = (c >> 3) * 16 + 4 * g + ((c >> 1) & 3);  // eight columns of a row a lane; rows 4-7 of a read are those of the upper half
    return KVTile<D, FP8>::place(r, 0) + 8 * (c & 1);
  } else {
    return KVTile<D, FP8>::place(4 * g + (c >> 2), (c >> 1) & 1) + 8 * (c & 1);  // four columns of a row a lane
  }
}
template <int D, bool FP8>
__device__ __forceinline__ bf16x8 kv_value_fragment(uint32_t first, int n) {
  if constexpr (FP8) {
    typedef __attribute__((ext_vector_type(2))) int i32x2;
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(uintptr_t)(first ^ (16 * n)));
    return widen((uint32_t)raw[0], (uint32_t)raw[1]);
  } else {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    constexpr int kUpper = KVTile<D, FP8>::kRow == 128 ? 16 : 0;  // the swizzle of row 16 + r differs in that
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(first ^ (32 * n)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((first ^ (32 * n) ^ kUpper) + 16 * KVTile<D, FP8>::kRow));
    typedef __attribute__((ext_vector_type(8))) short s16x8;
    return __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }
}

// Key of element e of a lane's eight, within the tile.
__device__ __forceinline__ int key_of(int g, int e) { return 16 * (e >> 2) + 4 * g + (e & 3); }

// Which of a lane's eight keys from key0 on a row of token tok sees: bit e. In the last tiles of a sequence only, so what a token sees is looked up anew there.
__device__ __forceinline__ uint32_t seen_keys(const KVAttnParams& p, const KVWork& s, int tok, int key0, int g) {
  const int ctx = s.len - s.n;  // rows in front of the new ones (below zero only where the lengths contradict each other)
  uint32_t seen = 0;
  if (p.tree) {
    const uint64_t word = (uint64_t)p.tree[s.tok0 + tok];
    const uint32_t lo = (uint32_t)word, hi = (uint32_t)(word >> 32);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = key0 + key_of(g, e), draft = key - ctx;
      const uint32_t bits = draft < 32 ? lo : hi;
      const int ok = ((draft < 0) | ((draft < 64) & (int)((bits >> (draft & 31)) & 1u))) & (int)(key < s.len);
      seen |= (uint32_t)ok << e;
    }
  } else {
    const int end = min(ctx + tok + 1, s.len);  // keys that the row sees
#pragma unroll
    for (int e = 0; e < 8; ++e) seen |= (uint32_t)(key0 + key_of(g, e) < end) << e;
  }
  return seen;
}

// Weights as the sum of two bf16 numbers, the upper 16 bits of each and the rounded rest of it: off by 2^-15 of the weight at most. The rest has 2^-20 of the weight on
// top, so that it is 0 only where the weight is: a value that is infinite stays so in the products with both. (Of infinite weights, which come of scales that are, the
// rest is NaN.)
__device__ __forceinline__ bf16x8 upper_halves(const float (&y)[8]) {
  u32x4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = __builtin_amdgcn_perm(__float_as_uint(y[2 * e + 1]), __float_as_uint(y[2 * e]), 0x07060302u);
  return __builtin_bit_cast(bf16x8, u);
}
__device__ __forceinline__ bf16x8 rests(const float (&y)[8]) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = fmaf(y[e], 1.f + 0x1p-20f, -__uint_as_float(__float_as_uint(y[e]) & 0xffff0000u));
  return to_bf16x8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
}

// Values that are not finite, in a tile that some rows see in part only: a row's weight of a key it does not see is 0, and must stay so against whatever the
// key's value holds. What such a value makes of a row that does see it is an infinity or NaN whatever the rest: `up` and `down` note, for each of the lane's
// features (bit 4 n + v), whether one above and one below all numbers was seen (NaN is both). Then it is 0 in LDS. Rare, and as slow as it likes to be.
template <int D, bool FP8, int R>
__device__ __forceinline__ void clean_values(char* values, int lane, const uint32_t (&seen)[R], uint32_t (&up)[R], uint32_t (&down)[R]) {
  using T = KVTile<D, FP8>;
  const auto finite = [](u32x4 x) __attribute__((always_inline)) {
    bool ok = true;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (FP8) ok = ok && ((x[k] & 0x7fu) != 0x7fu) & ((x[k] & 0x7f00u) != 0x7f00u) & ((x[k] & 0x7f0000u) != 0x7f0000u) & ((x[k] & 0x7f000000u) != 0x7f000000u);
      else ok = ok && ((x[k] & 0x7f80u) != 0x7f80u) & ((x[k] & 0x7f800000u) != 0x7f800000u);
    }
    return ok;
  };
  bool bad = false;
#pragma unroll
  for (int i = 0; i < T::kBytes / 1024; ++i) bad = bad || !finite(*reinterpret_cast<const u32x4*>(values + 16 * lane + 1024 * i));
  if (!__any(bad)) return;
  const int c = lane & 15, g = lane >> 4;
#pragma unroll 1
  for (int j = 0; j < kTileKeys; ++j) {
    const int owner = c + 16 * ((j >> 2) & 3), e = 4 * (j >> 4) + (j & 3);  // lane and element that hold key j of this lane's row
    uint32_t above = 0, below = 0;  // of the key's values
#pragma unroll 1
    for (int i = 0; i < D / 4; ++i) {
      const int d = 16 * (i >> 2) + 4 * g + (i & 3);
      bool inf, nan, negative;
      if constexpr (FP8) {  // (e4m3 has no infinities)
        const uint32_t x = *reinterpret_cast<const uint8_t*>(values + T::place(j, d >> 4) + (d & 15));
        inf = false, nan = (x & 0x7f) == 0x7f, negative = false;
      } else {
        const uint32_t x = *reinterpret_cast<const uint16_t*>(values + T::place(j, d >> 3) + 2 * (d & 7));
        inf = (x & 0x7fffu) == 0x7f80u, nan = (x & 0x7fffu) > 0x7f80u, negative = (x & 0x8000u) != 0;
      }
      above |= (uint32_t)(nan || (inf && !negative)) << i;
      below |= (uint32_t)(nan || (inf && negative)) << i;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool sees = (__shfl((int)seen[r], owner) >> e) & 1;
      up[r] |= sees ? above : 0;
      down[r] |= sees ? below : 0;
    }
  }
#pragma unroll 1
  for (int i = 0; i < T::kBytes / 1024; ++i) {
    u32x4* const at = reinterpret_cast<u32x4*>(values + 16 * lane + 1024 * i);
    u32x4 x = *at;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (FP8) {
#pragma unroll
        for (int b = 0; b < 32; b += 8)
          if (((x[k] >> b) & 0x7fu) == 0x7fu) x[k] &= ~(0xffu << b);
      } else {
        if ((x[k] & 0x7f80u) == 0x7f80u) x[k] &= 0xffff0000u;
        if ((x[k] & 0x7f800000u) == 0x7f800000u) x[k] &= 0xffffu;
      }
    }
    *at = x;
  }
}

// ---------------------------------------------------------------------------------------------

template <int D, bool FP8, int R>
__global__ __launch_bounds__(kKVThreads, (KVRing<D, FP8, R>::kPerUnit)) void kv_attn_kernel(KVAttnParams p) {
  using T = KVTile<D, FP8>;
  constexpr int kSlots = KVRing<D, FP8, R>::kSlots, kRing = KVRing<D, FP8, R>::kBytes;
  using Loads = KVLoads<D, FP8>;
  constexpr int M = 16 * R, kSteps = D / 32;  // of the score's contraction
  constexpr int kRegion = kRing > M * D * 4 ? kRing : M * D * 4;  // of a wave: its tiles, then its results
  __shared__ __attribute__((aligned(1024))) char lds[kKVWaves * kRegion];
  __shared__ __attribute__((aligned(1024))) char queries[KVQueries<D, R>::kBytes];
  __shared__ float2 wave_stats[kKVWaves][M];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  KVWalk<M> walk;
  if (!walk.start(p, lane)) return;
  char* const ring = lds + wave * kRegion;
  const int source = T::source(lane);
  const int key_at = T::place(c, g);  // of keys 0-15; 16-31 differ by this:
  constexpr int kUpperKey = 16 * T::kRow, kUpperXor = T::kRow == 256 ? 0 : 16;
  const int value_at = T::kBytes + kv_value_place<D, FP8>(c, g);

  do {
    const KVWork& s = walk.s;
    int head, row0;  // row0: within the sequence and head
    const int32_t* entries;
    if (p.head_tables > 1) {
      const int b = __builtin_amdgcn_readfirstlane(walk.seq / p.head_tables);
      head = walk.seq - b * p.head_tables;
      row0 = walk.block * M;
      entries = p.table + b * p.table_rs + head * p.table_hs;
    } else {
      const int per_head = (s.n * p.group + M - 1) / M;
      head = __builtin_amdgcn_readfirstlane(walk.block / per_head);
      const int i = walk.block - head * per_head;
      row0 = (i & 1 ? per_head - 1 - (i >> 1) : i >> 1) * M;  // first, last, second, last but one: of a prompt these see as much two by two
      entries = p.table + walk.seq * p.table_rs;
    }
    const int rows = min(s.n * p.group - row0, M);
    const int seen_by_any = p.tree ? s.len : min(max(s.len - s.n + __builtin_amdgcn_readfirstlane((row0 + rows - 1) / p.group) + 1, 0), s.len);  // keys that any row sees
    const ScalarTable table = (ScalarTable)(uintptr_t)entries;
    const int last = max(s.len - 1, 0);
    const int tile0 = walk.step * kKVWaves + wave;  // this wave's first
    const int tiles = min((seen_by_any + kTileKeys - 1) / kTileKeys, (walk.step + walk.n_steps()) * kKVWaves);
    const int n_tiles = tiles > tile0 ? (tiles - tile0 + kKVWaves - 1) / kKVWaves : 0;

    bf16x8 q[R][kSteps];
    int tok[R];
    f32x4 acc[R][D / 16];
    float m[R], l[R];  // reference and sum (this lane's keys) of a row
    uint32_t up[R], down[R];  // see clean_values
#pragma unroll
    for (int r = 0; r < R; ++r) {
      tok[r] = (row0 + min(16 * r + c, rows - 1)) / p.group;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) acc[r][n] = f32x4{};
      m[r] = -INFINITY;
      l[r] = 0.f;
      up[r] = down[r] = 0;
    }

    const auto key_of_tile = [&](int i) { return (tile0 + i * kKVWaves) * kTileKeys; };
    int pages[2];
    const auto look_up = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) pages[h] = table[min(key_of_tile(i) + 16 * h, last) >> p.cache.page_shift];
    };
    const auto request = [&](int i) __attribute__((always_inline)) {  // one of the first tiles
      look_up(i);
      const Loads loads(p, pages, key_of_tile(i), last, head);
      loads.keys(p, ring + i * T::kSlot, source, lane);
      loads.values(p, ring + i * T::kSlot, source);
    };
    // The queries stand in front of the first tiles in the queue.
    KVQueries<D, R>::stage(p, s, head, row0, rows, queries, wave, lane);
    const int ahead = min(kSlots, n_tiles);
#pragma unroll 1
    for (int i = 0; i < ahead; ++i) request(i);
    if (kSlots == 2 && ahead == 2) wait_loads<2 * T::kAll>();
    else if (ahead == 1) wait_loads<T::kAll>();
    else wait_loads<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();  // (the tiles stay under way)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {  // e4m3 keys are read 16 features at a time: steps 2 i, 2 i + 1 contract features 64 i + 16 g + {0..7, 8..15}
        const int piece = FP8 ? 8 * (i >> 1) + 2 * g + (i & 1) : 4 * i + g;
        q[r][i] = *reinterpret_cast<const bf16x8*>(queries + KVTile<D, false>::place(16 * r + c, piece));
      }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // the queries have been read
    asm volatile("" ::: "memory");
    if (n_tiles > 0) look_up(kSlots);
    int slot_at = 0;
#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
      char* const slot = ring + slot_at;
      const int key0 = key_of_tile(i);
      const int later = min(kSlots - 1, n_tiles - 1 - i);
      const bool more = i + kSlots < n_tiles;
      wait_tiles<D, FP8, kSlots, T::kLoads>(later);  // the keys
      f32x4 score[R][2];
      float k_scale[8], v_scale[8];
      {  // all fragments are asked for before the first product: an LDS read takes as long as several of them
        constexpr int kReads = FP8 ? kSteps / 2 : kSteps;  // of a half tile
        typename std::conditional<FP8, u32x4, bf16x8>::type raw[2][kReads];
        const uint32_t first = lds_address(slot) + key_at;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < kReads; ++j) raw[h][j] = *lds_at<typename std::conditional<FP8, u32x4, bf16x8>::type>((h == 0 ? first ^ (64 * j) : (first ^ kUpperXor ^ (64 * j)) + kUpperKey));
        f32x4 scales[4];
        if constexpr (FP8)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            scales[h] = *reinterpret_cast<const f32x4*>(slot + 2 * T::kBytes + 4 * (16 * h + 4 * g));
            scales[2 + h] = *reinterpret_cast<const f32x4*>(slot + 2 * T::kBytes + 128 + 4 * (16 * h + 4 * g));
          }
        if constexpr (R <= 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < R; ++r) score[r][h] = f32x4{};
#pragma unroll
          for (int j = 0; j < kReads; ++j) {
            if constexpr (FP8) {
              const bf16x8 k0 = widen(raw[h][j][0], raw[h][j][1]), k1 = widen(raw[h][j][2], raw[h][j][3]);
#pragma unroll
              for (int r = 0; r < R; ++r) score[r][h] = mfma16(k0, q[r][2 * j], score[r][h]);
#pragma unroll
              for (int r = 0; r < R; ++r) score[r][h] = mfma16(k1, q[r][2 * j + 1], score[r][h]);
            } else {
#pragma unroll
              for (int r = 0; r < R; ++r) score[r][h] = mfma16(raw[h][j], q[r][j], score[r][h]);
            }
          }
        }
        if constexpr (FP8)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int v = 0; v < 4; ++v) k_scale[4 * h + v] = scales[h][v] * p.kappa, v_scale[4 * h + v] = scales[2 + h][v];
      }
      const bool partial = key0 + kTileKeys > s.len - s.n + (p.tree ? 0 : 1);  // some row may not see all of it
      constexpr bool kSplit = R == 1;  // weights as two bf16 numbers
      bf16x8 weight[R];
      float unrounded[8];  // weights of the row, if they go in as two numbers
      uint32_t seen[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = score[r][e >> 2][e & 3] * (FP8 ? k_scale[e] : p.kappa);
        if (partial) {
          seen[r] = seen_keys(p, s, tok[r], key0, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = (seen[r] >> e) & 1 ? y[e] : -INFINITY;
        }
        float top = y[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, y[e]);
        if (__any(top > m[r] + kSlack)) {
          const float moved_to = moved(m[r], quad_max(top));
          const float alpha = moved_to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - moved_to);
          l[r] *= alpha;
#pragma unroll
          for (int n = 0; n < D / 16; ++n) scale_in_place(acc[r][n], alpha);
          m[r] = moved_to;
        }
        const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = __builtin_amdgcn_exp2f(y[e] - ref);
          l[r] += y[e];
        }
        if constexpr (FP8) {
          if (partial) {  // (the scale of a row that is not seen may hold anything)
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (seen[r] >> e) & 1 ? y[e] * v_scale[e] : 0.f;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= v_scale[e];
          }
        }
        if constexpr (kSplit) {
          weight[r] = upper_halves(y);
#pragma unroll
          for (int e = 0; e < 8; ++e) unrounded[e] = y[e];
        } else weight[r] = to_bf16x8(y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]);
        if constexpr (R > 2) __builtin_amdgcn_sched_barrier(0);
      }
      const Loads loads(p, pages, key_of_tile(i + kSlots), last, head);
      if (more) {  // (the keys have been read: their products have been used)
        loads.keys(p, slot, source, lane);
        look_up(i + kSlots + 1);
        wait_loads<(kSlots - 1) * T::kAll + T::kScaleLoads + T::kLoads>();
      } else {
        wait_tiles<D, FP8, kSlots, 0>(later);  // the values
      }
      if (partial) clean_values<D, FP8, R>(slot + T::kBytes, lane, seen, up, down);
      const uint32_t values = lds_address(slot) + value_at;
      constexpr int kAhead = R <= 2 ? D / 16 : 4;  // fragments asked for at once (64 rows: as registers allow)
#pragma unroll
      for (int n0 = 0; n0 < D / 16; n0 += kAhead) {
        bf16x8 v[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) v[n] = kv_value_fragment<D, FP8>(values, n0 + n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r][n0 + n] = mfma16(v[n], weight[r], acc[r][n0 + n]);
        if constexpr (kSplit) {
          __builtin_amdgcn_sched_barrier(0);
          const bf16x8 rest = rests(unrounded);
#pragma unroll
          for (int n = 0; n < kAhead; ++n) acc[0][n0 + n] = mfma16(v[n], rest, acc[0][n0 + n]);
        }
      }
      if (more) {
        __builtin_amdgcn_s_waitcnt(0xC07F);  // the values have been read
        asm volatile("" ::: "memory");
        loads.values(p, slot, source);
      }
      slot_at = slot_at + T::kSlot == kRing ? 0 : slot_at + T::kSlot;
    }

    // The waves' results of the segment, joined through LDS: a wave's rows lie in its own region, piece (four features) q of row r at q ^ (r % 16).
    constexpr int kRowPieces = D / 4;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      l[r] = quad_sum(l[r]);
      if (g == 0) wave_stats[wave][16 * r + c] = make_float2(m[r], l[r]);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kKVWaves; ++w) top = fmaxf(top, wave_stats[w][16 * r + c].x);
      const float f = __builtin_amdgcn_exp2f(m[r] - (top == -INFINITY ? 0.f : top));
#pragma unroll
      for (int n = 0; n < D / 16; ++n) *reinterpret_cast<f32x4*>(ring + ((16 * r + c) * kRowPieces + ((4 * n + g) ^ c)) * 16) = acc[r][n] * f;
      if (__any((up[r] | down[r]) != 0))
#pragma unroll 1
        for (int i = 0; i < D / 4; ++i)
          if (((up[r] | down[r]) >> i) & 1)
            *reinterpret_cast<float*>(ring + ((16 * r + c) * kRowPieces + ((4 * (i >> 2) + g) ^ c)) * 16 + 4 * (i & 3)) =
                !((down[r] >> i) & 1) ? INFINITY : (up[r] >> i) & 1 ? NAN : -INFINITY;
    }
    __syncthreads();
    const bool whole = walk.whole(p);
    const int64_t slot = walk.slot(p);
    for (int i = threadIdx.x; i < rows * kRowPieces; i += kKVThreads) {
      const int row = i / kRowPieces, piece = i % kRowPieces;
      float top = -INFINITY, sum = 0.f;
      float2 st[kKVWaves];
#pragma unroll
      for (int w = 0; w < kKVWaves; ++w) st[w] = wave_stats[w][row], top = fmaxf(top, st[w].x);
      const float ref = top == -INFINITY ? 0.f : top;
      f32x4 x = {};
#pragma unroll
      for (int w = 0; w < kKVWaves; ++w) {
        x += *reinterpret_cast<const f32x4*>(lds + w * kRegion + (row * kRowPieces + (piece ^ (row & 15))) * 16);
        sum += st[w].y * __builtin_amdgcn_exp2f(st[w].x - ref);  // (a wave that saw nothing: 0; one that saw NaN only: NaN)
      }
      if (whole) {
        const int tok = (row0 + row) / p.group, h = head * p.group + row0 + row - tok * p.group;
        const int64_t t = s.tok0 + tok;
        const f32x4 o = sum == 0.f ? f32x4{} : x * (1.f / sum);
        *reinterpret_cast<u32x2*>(p.o + t * p.o_ts + h * p.o_hs + 4 * piece) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
        if (piece == 0) p.lse[h * p.lse_hs + t] = sum == 0.f ? -INFINITY : ref + __builtin_amdgcn_logf(sum);
      } else {
        *reinterpret_cast<f32x4*>(p.results + (slot * M + row) * D + 4 * piece) = x;
        if (piece == 0) p.stats[slot * M + row] = make_float2(top, sum);
      }
    }
    walk.leave_join(p, row0, head, rows);
    __syncthreads();  // the rings are free
  } while (walk.next(p));
}

template <int D>
void launch_kv_attn(const KVAttnParams& p, bool fp8, int row_groups, int workgroups, hipStream_t s) {
  if constexpr (D == 128)
    if (row_groups == 4) {  // (bf16 only, see plan_of)
      kv_attn_kernel<128, false, 4><<<workgroups, kKVThreads, 0, s>>>(p);
      return;
    }
  const auto launch = [&](auto f) {
    constexpr bool F = decltype(f)::value;
    if (row_groups == 1) kv_attn_kernel<D, F, 1><<<workgroups, kKVThreads, 0, s>>>(p);
    else kv_attn_kernel<D, F, 2><<<workgroups, kKVThreads, 0, s>>>(p);
  };
  if (fp8) launch(std::true_type());
  else launch(std::false_type());
}
void launch_kv_attn_d128(const KVAttnParams& p, bool fp8, int row_groups, int workgroups, hipStream_t s);  // kv_attn.hip
void launch_kv_attn_d64(const KVAttnParams& p, bool fp8, int row_groups, int workgroups, hipStream_t s);   // kv_attn_d64.hip

}  // namespace pith
