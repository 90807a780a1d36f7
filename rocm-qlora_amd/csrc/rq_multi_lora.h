// Kernels shared by the adapters' forward and backward passes over grouped rows
// (rq_rows.h).  An adapter's factors are A [r, K] and B [N, r] in the rows' dtype.
//
//   shrink   part[split][slot][j] = sum over a split's k of x[row][k] S[j][k]
//   expand   out[row][c] = base[row][c] + scale * sum_j u[slot][j] S[c, j], u the splits' sum
//            (and u as the operands that rowsum reads)
//   operands those operands alone
//   rowsum   D[c][j] = scale * sum over an adapter's rows of x[row][c] u[slot][j]
//
// 16-bit rows: u is an fp32 sum, and the matrix instructions take 16-bit operands.
// It is passed as two of them, hi = RND(u) and lo = RND(u - hi), whose products
// are both added: 16 bits of u (bf16; 22 fp16) instead of 8 (11), at twice the
// products over the rank alone, which memory hides.  fp16 has lo times 2^11, undone
// in the fp32 sums (a training step of 4096 rows, r 64: 3 us of 170), so that a small u
// (a gradient's g = dY B while B is near zero) keeps 22 bits down to 2^-14 and a
// resolution of 2^-36 below, instead of 2^-25.  fp32 rows run on the fp32
// matrix instructions.  So fp16 rows take u up to 65504, as a first product rounded
// to fp16 would, and an infinity in B, or in a gradient's x or dY, may come out as NaN
// (infinity times a lo part of zero); what is not finite never comes out finite.
#pragma once

#include "rq_io.h"
#include "rq_rows.h"

namespace rq {

// Ranks stored for a slot (zeros past r): 16, whose hi and lo parts share one 32-deep
// matrix instruction, or a multiple of 32.
inline int64_t rank_pad(int64_t r) { return r <= 16 ? 16 : ceil_div(r, 32) * 32; }

struct ShrinkArgs {
  RowsPlan rows;
  const void* x;
  int64_t ldx, K;
  const void* s;        // factor of adapter a at s + a * s_adapter
  int64_t s_adapter;
  int r, rp;
  int splits;
  int64_t k_per_split;  // a multiple of the waves' steps
  float* part;          // [splits][slots][rp]
};

struct ExpandArgs {
  RowsPlan rows;
  const float* part;    // [splits][slots][rp]
  int splits;
  int r, rp;
  const void* s;        // factor of adapter a at s + a * s_adapter
  int64_t s_adapter;
  int64_t C;            // columns of out
  const float* scaling; // [n]
  const void* base;     // [M][ld_base], or nullptr: zeros
  int64_t ld_base;
  void* out;
  int64_t ld_out;
  void* opt;            // rowsum's operands of the splits' sum, or nullptr
  int chunks, iters;    // column chunks of a tile, steps of a wave in each
};

struct OperandsArgs {
  RowsPlan rows;
  int r, rp;
  const float* part;    // [splits][slots][rp]
  int splits;
  void* opt;            // slots * rp values of 32 bits
};

// The row sums' operands in the order in which rowsum's lanes load them: for 32 slots and 16
// ranks, 1 KiB of hi parts and 1 KiB of lo parts (fp32: of slots 8 g .. 8 g + 3 and of the four
// after them), 16 bytes of lane (i, g) = rank i, slots 8 g .. 8 g + 7.  slot: a multiple of 8.
template <int XT>
__host__ __device__ inline int64_t opt_at(int64_t slot, int rank, int rp) {
  constexpr int kBlock = XT == RQ_DTYPE_F32 ? 512 : 1024, kLane = Elem<XT>::kVec;
  return ((slot >> 5) * (rp >> 4) + (rank >> 4)) * kBlock + ((rank & 15) + 2 * (slot & 24)) * kLane;
}

// 16-rank blocks of a rowsum wave: 1, 2 or 4.
__host__ __device__ inline int rowsum_blocks(int rp) { return rp <= 16 ? 1 : (rp <= 32 ? 2 : 4); }

// First rank of the operands that block j of the wave from rank j0 on loads: its own, or where
// the stored ranks end before it (rp 96: blocks 6 and 7) the wave's first again, whose sums are
// not stored.
__host__ __device__ inline int rowsum_rank(int j0, int j, int rp) { return j0 + 16 * j < rp ? j0 + 16 * j : j0; }

struct RowSumTask {
  const void* src;      // rows, or 8-bit codes
  const uint8_t* exps;  // of the codes, or nullptr: src holds values
  int64_t ld;           // elements (codes) per row
  int64_t C;            // columns
  const void* opt;      // operands of u
  void* out;            // [n][C][r], or [n][r][C] when rank_major
  bool rank_major;
  int64_t part_off;     // of this task's values in a partial slot
  int tiles;            // column tiles
};

struct RowSumArgs {
  RowsPlan rows;
  int table;            // chunk table of the plan
  int r, rp;
  const float* scaling; // [n]
  RowSumTask t[2];
  int n;
  float* part;          // [parts][part_size]
  int64_t part_size;
};

}  // namespace rq
