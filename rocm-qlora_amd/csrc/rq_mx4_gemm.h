// What the matrix products on MXFP4 weights share (mx4_gemm.hip, mx4_a4.hip): arguments, the
// output of a wave's block, the K splits' sum.
#pragma once

#include "rq_gemm_core.h"
#include "rq_mx4.h"

namespace rq {

constexpr int kMgThreads = 512;
constexpr int kMgStep = 64;

struct MxGemmArgs {
  const uint8_t* x;    // 16-bit rows, 16-byte aligned, zeros up to whole steps
  int64_t ldx;         // bytes
  int64_t plane;       // bytes between the planes of split fp32 rows
  int planes;
  int xdiv;
  bool by_slot;        // rows of x are the plan's slots
  RowsPlan rows;
  const uint8_t* codes;
  const uint8_t* scales;  // forward: bytes [E][wrows][pitch / 16]; dX: bf16 [E][pitch / 16][np]
  int64_t wrows, pitch;   // the weight's rows and bytes of a row's codes
  int64_t np;             // dX: wrows rounded up to steps
  int64_t cols;           // of the output
  int nk;                 // steps of a plane
  int splits;
  int row_tiles, col_tiles;
  const void* bias;    // [E][cols]
  int bias_dt;
  void* y;             // 16-bit rows, or fp32 [splits][M][ldy]
  int64_t ldy;
};

// LDS that direct-to-LDS loads alone write: the compiler sees no store to it, and would take what
// is read there for undefined.
__device__ __forceinline__ void lds_escapes(uint8_t* lds) {
  asm volatile("" ::"v"((__attribute__((address_space(3))) uint8_t*)lds) : "memory");
}

// Bytes of a wave's staged row of 32 NB 16-bit outputs.
__host__ __device__ constexpr int mx_out_pitch(int NB) { return 64 * NB + 16; }

// The results of a wave: 32 MB rows from slot0 + rw, columns cw ...  `stage`: 32 MB mx_out_pitch(NB) bytes of
// LDS of its own (16-bit results).
//
// Output.  Block (mb, nb): lane (i32, q) holds row 32 mb + i32 of the wave's, and in register r the
// A operand's row 8 (r / 4) + 4 q + r % 4: forward column 32 nb + that, dX 4 that + nb.  Four values
// v of adjacent columns: forward registers 4 h .. of block nb, dX register r of the four blocks.
template <int XT, bool DX, int MB, int NB, bool OUT32>
__device__ __forceinline__ void mx_output(const MxGemmArgs& a, const f32x16 (&acc)[MB][NB], uint8_t* stage, int lane, int64_t e,
                                          bool live, int split, int64_t slot0, int count, int rw, int64_t cw) {
  constexpr int kOutPitch = mx_out_pitch(NB);
  const int i32 = lane & 31, q = lane >> 5;
  constexpr int kQuads = DX ? 16 : 4 * NB;
  auto quad = [&](int mb, int k, float (&v)[4]) -> int {  // returns the first column, of the wave's
    if constexpr (DX) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = acc[mb][c][k];
      return 4 * (8 * (k / 4) + 4 * q + k % 4);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = acc[mb][k / 4][4 * (k % 4) + c];
      return 32 * (k / 4) + 8 * (k % 4) + 4 * q;
    }
  };
  const bool biased = a.bias && live && split == 0;
#pragma unroll
  for (int k = 0; k < kQuads; ++k) {
    float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (biased) {
      const int64_t col = cw + (DX ? 0 : 32 * (k / 4) + 8 * (k % 4) + 4 * q);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (col + c < a.cols) bias[c] = load_as_f32(a.bias, e * a.cols + col + c, a.bias_dt);
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      float v[4];
      const int col = quad(mb, k, v);
      if (biased) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = __fadd_rn(v[c], bias[c]);
      }
      const int r = rw + 32 * mb + i32;
      if constexpr (OUT32) {
        if (r >= count) continue;
        float* p = static_cast<float*>(a.y) + (int64_t(split) * a.rows.M + plan_row(a.rows, slot0 + r)) * a.ldy + cw + col;
        const int64_t left = a.cols - cw - col;
        if (left >= 4) store16_any(p, u32x4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])});
        else
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < left) p[c] = v[c];
      } else {
        *reinterpret_cast<u32x2*>(stage + (32 * mb + i32) * kOutPitch + 2 * col) =
            u32x2{cvt_pk<XT>(v[0], v[1]), cvt_pk<XT>(v[2], v[3])};
      }
    }
  }
  if constexpr (!OUT32) {
    // the wave reads back its own rows, 16 bytes a lane
    constexpr int kLanes = 4 * NB;  // of a row
#pragma unroll 4
    for (int it = 0; it < 32 * MB * kLanes / 64; ++it) {
      const int r = it * (64 / kLanes) + lane / kLanes, c = lane % kLanes;
      if (rw + r >= count) continue;
      const u32x4 v = *reinterpret_cast<const u32x4*>(stage + r * kOutPitch + 16 * c);
      const int64_t col = cw + 8 * c, row = plan_row(a.rows, slot0 + rw + r);
      uint16_t* p = static_cast<uint16_t*>(a.y) + row * a.ldy + col;
      const int64_t left = a.cols - col;
      if (left >= 8) store16_any(p, v);
      else if (left > 0) store_edge<XT>(p, v, int(left));
    }
  }
}

// Adds up partial sums [splits][M][ld] (mx4_gemm.hip).
struct MxSumArgs {
  const float* part;
  int64_t M, ld;
  int splits, ysum;
  int64_t out_rows, cols;
  void* y;
  int64_t ldy;
};
void mx4_sum(const MxSumArgs& s, int dt, hipStream_t stream);

inline int64_t up256(int64_t n) { return (n + 255) & ~int64_t(255); }

}  // namespace rq
