// Packed (ragged) attention: what the kernels and the entry point share.
#pragma once

#include "kernels.cuh"

namespace vcattn {

// One unit of work of a packed batch (32 bytes; vcattn_packed_tile in the C
// ABI).  Rows are the sequence's (token, group head) pairs, row = token * G +
// g, or its tokens, depending on the kernel.
struct PackedTile {
  int q0, lq;   // first query row of the sequence in the packed buffer, queries
  int k0, lk;   // same for the keys
  int r0;       // first row of this tile
  int kb, ke;   // keys [kb, ke) of the sequence (empty: the output rows are 0)
  int slot;     // index of its partial result, or -1: writes the output itself
};

// A group of partial results that join into one tile's output rows.
struct PackedJoin {
  int q0, lq, r0;
  int slot0, pieces;
  int unused[3];
};

// Arguments of one kernel over one list of tiles.
struct PackedArgs {
  const void *q, *k, *v;
  void* out;
  int64_t qsh, qsn, ksh, ksn, vsh, vsn, osh, osn;   // strides in elements over heads and rows
  const PackedTile* tiles;
  const PackedJoin* joins;
  int n_tiles, n_joins, slots;
  int Hq, Hk, G, D;
  int Tq, Tk;      // rows of the packed buffers: no tile reads or writes past them
  int causal;
  float scale_log2;   // softmax scale * log2(e)
  float* part_o;      // [slot][head][rows][D]
  float* part_ml;     // [slot][head][rows][2]: reference (log2 domain) and sum
};

// Rows of a tile, and so of a partial result, of the three lists of a batch:
// (token, group head) pairs of one KV head on register MMAs, tokens of one
// query head on tcgen05.
constexpr int kPackedFewRows = 16;
constexpr int kPackedRows = 64;
constexpr int kPackedWideRows = 256;
constexpr int kListRows[3] = {kPackedFewRows, kPackedRows, kPackedWideRows};

// A record as the kernels use it: empty (no row, no key) if it points before the
// buffers or outside the workspace, or if its row and key numbers leave 31 bits
// (rows and keys past Tq and Tk are left out where they are read and written).
__device__ __forceinline__ bool fits31(int64_t n) { return n < (int64_t{1} << 31) - kPackedWideRows; }
__device__ __forceinline__ PackedTile load_tile(const PackedArgs& a, int i, int group) {
  PackedTile t = a.tiles[i];
  const int64_t rows = static_cast<int64_t>(t.lq) * group;
  if ((t.q0 | t.lq | t.k0 | t.lk | t.r0 | t.kb) < 0 || t.slot >= a.slots || t.r0 >= rows || !fits31(rows) ||
      !fits31(static_cast<int64_t>(t.q0) + t.lq) || !fits31(static_cast<int64_t>(t.k0) + t.lk))
    return PackedTile{0, 0, 0, 0, 0, 0, 0, -1};
  t.ke = min(t.ke, min(t.lk, max(0, a.Tk - t.k0)));
  return t;
}
__device__ __forceinline__ PackedJoin load_join(const PackedArgs& a, int i, int group) {
  const PackedJoin j = a.joins[i];
  if ((j.q0 | j.lq | j.r0 | j.slot0 | j.pieces) < 0 || static_cast<int64_t>(j.slot0) + j.pieces > a.slots ||
      !fits31(static_cast<int64_t>(j.lq) * group) || j.r0 >= static_cast<int64_t>(j.lq) * group ||
      !fits31(static_cast<int64_t>(j.q0) + j.lq))
    return PackedJoin{0, 0, 0, 0, 0, {0, 0, 0}};
  return j;
}

cudaError_t launch_attn_packed_tc(const PackedArgs& a, int dtype, cudaStream_t st);

}  // namespace vcattn
