// The rows of a batch grouped by adapter.
//
// Rows are laid out in tiles of 64 slots, each tile of one adapter: the rows of
// adapter 0 in their order, padded to whole tiles, then adapter 1's, .., then the
// rows without an adapter.  What is computed per row between two launches (the
// rank-wide operands) is stored by slot, so that a tile's rows are adjacent
// whatever their order in the batch.  Sums over an adapter's rows run over chunks
// of its tiles; an adapter of one chunk (or of no row) writes its result at once, the
// others' partial sums are added in order.  There are two tables of chunks, of 4 and of
// 16 tiles at least: few columns take the finer one.
//
// The plan is int32 device memory:
//   [0] tiles in use, [1], [2] chunks in use of the two tables, [3], [4] big tiles in use of the two
//   tables, [5..15] zero
//   tile[T][2]                        (adapter, -1: rows without one; rows, 0: not in use)
//   slot_row[64 T]                    (-1: padding; of tiles in use)
//   chunk[2][C][4]                    (adapter, first tile, end tile, partial slot or -1)
//   part[2][n][2]                     (chunks of the adapter, its first partial slot)
//   big[2][S]                         (first tile of each two, four adjacent tiles of an adapter, or what
//                                      is left of its tiles; rows without one last)
// A null plan stands for M rows of adapter 0 in their own order.
#pragma once

#include "rq_common.h"

namespace rq {

constexpr int kTileRows = 64;
constexpr int kMaxAdapters = 1024;
// Tiles of a chunk, before an adapter's chunks are made alike: at least these, and at least 1 / kRowChunks of all, so that
// partial sums are bounded: adapters of several chunks have at most 2 kRowChunks of
// them in all.
constexpr int kRowChunks = 16;
constexpr int kChunkTables = 2;
__host__ __device__ constexpr int chunk_least(int table) { return table == 0 ? 4 : 16; }
constexpr int kMaxParts = 2 * kRowChunks;
constexpr int kBigTables = 2;
__host__ __device__ constexpr int big_tiles(int table) { return 2 << table; }  // tiles of a big one

struct RowsPlan {
  const int32_t* p;  // device, or nullptr
  int64_t M;
  int32_t n;         // adapters
  int32_t T;         // tiles, at most
  int32_t C;         // chunks of a table, at most

  __host__ __device__ int64_t off_rows() const { return 16 + ((2 * int64_t(T) + 3) & ~int64_t(3)); }
  __host__ __device__ int64_t off_chunks() const { return off_rows() + int64_t(kTileRows) * T; }
  __host__ __device__ int64_t off_part() const { return off_chunks() + kChunkTables * 4 * int64_t(C); }
  __host__ __device__ int64_t off_big() const { return off_part() + kChunkTables * 2 * int64_t(n); }
  // big tiles of a table, at most: whole ones and an end of each adapter's
  __host__ __device__ int64_t bigs(int table) const {
    const int64_t some = int64_t(n) + 1 < T ? int64_t(n) + 1 : T;
    return T / big_tiles(table) + some;
  }
  __host__ __device__ int64_t words() const { return off_big() + bigs(0) + bigs(1); }
  __host__ __device__ int64_t slots() const { return int64_t(kTileRows) * T; }

  // tiles per chunk when `tiles` are in use
  __host__ __device__ static int chunk_tiles(int tiles, int table) {
    const int c = (tiles + kRowChunks - 1) / kRowChunks;
    return c > chunk_least(table) ? c : chunk_least(table);
  }
};

// An adapter's chunks: as few as chunk_tiles allows, of the same size but for the last.
struct Chunks {
  int n, tiles;
};
__host__ __device__ inline Chunks adapter_chunks(int tiles, int all, int table) {
  const int most = RowsPlan::chunk_tiles(all, table), n = tiles > most ? (tiles + most - 1) / most : 1;
  return Chunks{n, (tiles + n - 1) / n};
}

// A tile's adapter and rows in use, as every workgroup of the tile reads them.
struct Tile {
  int adapter;
  int count;  // 0: the tile is not in use
};

__device__ __forceinline__ Tile plan_tile(const RowsPlan& P, int t) {
  if (!P.p) {
    const int64_t left = P.M - int64_t(kTileRows) * t;
    return Tile{0, left < kTileRows ? int(left > 0 ? left : 0) : kTileRows};
  }
  const u32x2 v = *reinterpret_cast<const u32x2*>(P.p + 16 + 2 * int64_t(t));
  return Tile{int(v.x), int(v.y)};
}

// The slot's row, -1 for padding (slots of tiles not in use: anything).
__device__ __forceinline__ int plan_row(const RowsPlan& P, int64_t slot) {
  if (!P.p) return slot < P.M ? int(slot) : -1;
  return P.p[P.off_rows() + slot];
}

// Host: the largest tile and chunk counts of M rows and n adapters.
inline RowsPlan rows_plan(const int32_t* p, int64_t M, int64_t n) {
  const int64_t some = n + 1 < M ? n + 1 : M;
  RowsPlan P{p, M, int32_t(n), 0, 0};
  P.T = int32_t(p ? M / kTileRows + some : ceil_div(M, kTileRows));
  P.C = int32_t(p ? n + kMaxParts : ceil_div(P.T, RowsPlan::chunk_tiles(P.T, 0)));
  return P;
}

}  // namespace rq
