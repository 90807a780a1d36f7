// Kernels shared by the adapters' forward and backward passes over grouped rows
// (rq_rows.h).  An adapter's factors are A [r, K] and B [N, r] in the rows' dtype.
//
//   shrink   part[split][slot][j] = sum over a split's k of x[row][k] S[j][k]
//   finish   the splits' sum, in order, as fp32 and as what the products below read
//   expand   out[row][c] = base[row][c] + scale * sum_j u[slot][j] S[c, j]
//   rowsum   D[c][j] = sum over an adapter's rows of x[row][c] u[slot][j]
//
// 16-bit rows: u is an fp32 sum, and the matrix instructions take 16-bit operands.
// It is passed as two of them, hi = RND(u) and lo = RND(u - hi), whose products
// are both added: 16 bits of u (bf16; 22 fp16) instead of 8 (11), at twice the
// products over the rank alone, which memory hides.  fp32 rows run on the fp32
// matrix instructions.
#pragma once

#include "rq_io.h"
#include "rq_rows.h"

namespace rq {

// ranks stored for a slot: r rounded up to 16
inline int64_t rank16(int64_t r) { return ceil_div(r, 16) * 16; }

struct ShrinkArgs {
  RowsPlan rows;
  const void* x;
  int64_t ldx, K;
  const void* s;        // [n][.][ld_s]
  int64_t ld_s, s_adapter;
  int r;                // live rows of s
  int r16;
  int splits;
  int64_t k_per_split;  // a multiple of 4 waves' steps
  float* part;          // [splits][slots][r16]
};

struct FinishJob {
  const float* part;    // [splits][slots][r16]
  int splits;
  bool scaled;          // times the adapter's scaling
  float* sum;           // [slots][r16] fp32, or nullptr
  void* op;             // 16-bit: [slots][2 r16], hi | lo; fp32: [slots][r16]; or nullptr
  void* opt;            // 16-bit: [2][r16][slots]; fp32: [r16][slots]; or nullptr
};

struct FinishArgs {
  RowsPlan rows;
  int r16;
  const float* scaling;
  FinishJob job[2];
  int jobs;
};

struct ExpandArgs {
  RowsPlan rows;
  const void* op;       // finish's
  int r, r16;
  const void* s;        // factor of adapter a at s + a * s_adapter
  int64_t s_adapter, ld_s;
  int64_t C;            // columns of out
  const float* scaling; // per adapter, or nullptr: 1
  const void* base;     // [M][ld_base], or nullptr: zeros
  int64_t ld_base;
  void* out;
  int64_t ld_out;
  int chunks;           // column chunks of a workgroup
};

struct RowSumTask {
  const void* src;      // rows, or 8-bit codes
  const uint8_t* exps;  // of the codes, or nullptr: src holds values
  int64_t ld;           // elements (codes) per row
  int64_t C;            // columns
  const void* opt;      // finish's
  void* out;            // [n][C][r], or [n][r][C] when rank_major
  bool rank_major;
  int64_t part_off;     // of this task's values in a partial slot
  int tiles;            // column tiles
};

struct RowSumArgs {
  RowsPlan rows;
  int r, r16;
  RowSumTask t[2];
  int n;
  float* part;          // [kMaxParts][part_size]
  int64_t part_size;
};

// columns of a lane of the row sums, by 16-rank blocks of a workgroup
template <int XT>
constexpr int rowsum_cw(int jb) {
  return XT == RQ_DTYPE_F32 || jb > 2 ? 4 : 8;
}
template <int XT>
constexpr int expand_cols() { return 16 * Elem<XT>::kVec; }  // of a wave

template <int XT>
int run_shrink(const ShrinkArgs& a, hipStream_t stream);
template <int XT>
int run_finish(const FinishArgs& a, hipStream_t stream);
// FACTOR_ROWS: S[c, j] at s[c * ld_s + j] (B); otherwise at s[j * ld_s + c] (A).
template <int XT, bool FACTOR_ROWS>
int run_expand(ExpandArgs a, hipStream_t stream);
template <int XT>
int run_rowsum(RowSumArgs a, hipStream_t stream);

// Splits of a shrink over K and their length, for `cus` compute units.
void plan_shrink(int64_t T, int64_t K, int step, int cus, int* splits, int64_t* per);

}  // namespace rq
