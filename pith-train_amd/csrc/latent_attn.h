// Attention to the latent cache: what its kernels share. The work list, the tiles and the join.
//
// Work list. A sequence of n new tokens and L rows is ceil(n H / M) row blocks (row = token * H + head; M of them share a workgroup's tiles) times
// ceil(L / 64) tiles of 64 keys, and the tiles of all row blocks of all sequences, one behind the other, are dealt to the workgroups in equal
// ranges. Lengths are read on the device, so nothing depends on the host knowing them: a captured call follows its sequences as they grow, and one
// long sequence among short ones is spread over as many workgroups as its share of the tiles. A workgroup whose range covers a row block wholly
// writes its rows; parts of a row block leave (sum, maximum, unnormalised result) in fp32 in the workspace, and a second kernel joins them in the
// order of the keys (results do not depend on scheduling).
#pragma once

#include "attn_tiles.h"
#include "latent_common.h"

namespace pith {

constexpr int kLatentKeys = 64;  // keys of a tile

// load_lds16 from an address of each lane's own.
__device__ __forceinline__ void load_lds16_at(const void* src, char* dst_wave) {
  const uint32_t lds_addr = (uint32_t)(uintptr_t)(lds_char*)dst_wave;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(src) : "memory");
}

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
  int* items;    // number of row blocks of this call
  int4* joins;   // [row blocks] what the join needs of each: first row (token * H + head of the whole call), rows, first and last slot (equal: nothing)
  float2* stats; // [slots][M] running maximum (in bits) and sum
  float* parts;  // [slots][M][512]
  int max_items; // capacity of joins
  int min_tiles; // of a workgroup's range
};

struct SeqWork {
  int tok0, n, len;       // first token, new tokens, cached rows
  int blocks, tiles;      // row blocks, tiles of each
};

__device__ __forceinline__ SeqWork seq_work(const LatentAttnParams& p, int b, int rows_per_block) {
  SeqWork s;
  const int c0 = min(max(p.cu_q[b], 0), p.T), c1 = min(max(p.cu_q[b + 1], c0), p.T);
  s.tok0 = c0;
  s.n = c1 - c0;
  s.len = min(max(p.lengths[b], 0), p.max_len);
  s.blocks = (s.n * p.H + rows_per_block - 1) / rows_per_block;
  s.tiles = max((s.len + kLatentKeys - 1) / kLatentKeys, 1);  // rows without keys get their zeros from an empty tile
  return s;
}

// Inclusive sums over the lanes of a wavefront.
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    x += lane >= d ? y : 0;
  }
  return x;
}

}  // namespace pith
