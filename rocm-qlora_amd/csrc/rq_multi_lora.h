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
// products over the rank alone, which memory hides.  fp32 rows run on the fp32
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
