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
  int cus;             // compute units
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

// Bytes of a wave's staged row of 32 NB outputs, and of what it stages at once: its 32 MB rows, of fp32 results 32.
__host__ __device__ constexpr int mx_out_pitch(int NB, bool out32) { return (out32 ? 128 : 64) * NB + 16; }
__host__ __device__ constexpr int mx_out_wave(int MB, int NB) {
  const int a = 32 * MB * mx_out_pitch(NB, false), b = 32 * mx_out_pitch(NB, true);
  return a > b ? a : b;
}

// The results of a wave: 32 MB rows from slot0 + rw, columns cw ...  `stage`: mx_out_wave(MB, NB) bytes of
// LDS of its own.  Block (mb, nb): lane (i32, q) holds row 32 mb + i32 of the wave's, and in register r the
// A operand's row 8 (r / 4) + 4 q + r % 4: forward column 32 nb + that, dX 4 that + nb; so four values of
// adjacent columns are forward registers 4 h .. of block nb, dX register r of the four blocks.  (fp32 results
// stored straight from registers, 16 bytes a row, took twice the time.)
template <int XT, bool DX, int MB, int NB, bool OUT32>
__device__ __forceinline__ void mx_output(const MxGemmArgs& a, const f32x16 (&acc)[MB][NB], uint8_t* stage, int lane, int64_t e,
                                          bool live, int split, int64_t slot0, int count, int rw, int64_t cw) {
  constexpr int kPitch = mx_out_pitch(NB, OUT32);
  const int i32 = lane & 31, q = lane >> 5;
  // (never with dX; past the columns zeros)
  const bool biased = !DX && a.bias && live && split == 0 && cw < a.cols;
  const int bs = a.bias_dt == RQ_DTYPE_F32 ? 4 : 2;
  const __amdgpu_buffer_rsrc_t br =
      buffer_rsrc(static_cast<const uint8_t*>(a.bias) + (biased ? (e * a.cols + cw) * bs : 0),
                  biased ? uint32_t((a.cols - cw < 32 * NB ? a.cols - cw : 32 * NB) * bs) : 0u);
  constexpr int kQuads = DX ? 16 : 4 * NB;
  constexpr int ES = OUT32 ? 4 : 2, V = 16 / ES;
  constexpr int kOnce = OUT32 ? 1 : MB;  // 32-row blocks staged at a time
#pragma unroll
  for (int m0 = 0; m0 < MB; m0 += kOnce) {
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const int col = DX ? 4 * (8 * (k / 4) + 4 * q + k % 4) : 32 * (k / 4) + 8 * (k % 4) + 4 * q;  // the quad's first
      float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (biased) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t at = uint32_t(col + c);
          if (a.bias_dt == RQ_DTYPE_F32) bias[c] = u2f(buf_load4(br, 4 * at));
          else if (a.bias_dt == RQ_DTYPE_BF16) bias[c] = bf16_to_f32(uint16_t(buf_load2(br, 2 * at)));
          else bias[c] = f16_to_f32(uint16_t(buf_load2(br, 2 * at)));
        }
      }
#pragma unroll
      for (int m = 0; m < kOnce; ++m) {
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if constexpr (DX) v[c] = acc[m0 + m][c][k];
          else v[c] = __fadd_rn(acc[m0 + m][k / 4][4 * (k % 4) + c], bias[c]);
        }
        uint8_t* o = stage + (32 * m + i32) * kPitch + ES * col;
        if constexpr (OUT32) *reinterpret_cast<u32x4*>(o) = u32x4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
        else *reinterpret_cast<u32x2*>(o) = u32x2{cvt_pk<XT>(v[0], v[1]), cvt_pk<XT>(v[2], v[3])};
      }
    }
    // the wave reads back its own rows, 16 bytes a lane
    constexpr int kLanes = 32 * NB / V;  // of a row
#pragma unroll 4
    for (int it = 0; it < 32 * kOnce * kLanes / 64; ++it) {
      const int at = it * 64 + lane, r = at / kLanes, c = at % kLanes;
      if (rw + 32 * m0 + r >= count) continue;
      const u32x4 v = *reinterpret_cast<const u32x4*>(stage + r * kPitch + 16 * c);
      const int64_t col = cw + V * c, row = plan_row(a.rows, slot0 + rw + 32 * m0 + r);
      const int64_t left = a.cols - col;
      if constexpr (OUT32) {
        float* p = static_cast<float*>(a.y) + (int64_t(split) * a.rows.M + row) * a.ldy + col;
        if (left >= 4) store16_any(p, v);
        else if (left > 0) store_edge<RQ_DTYPE_F32>(p, v, int(left));
      } else {
        uint16_t* p = static_cast<uint16_t*>(a.y) + row * a.ldy + col;
        if (left >= 8) store16_any(p, v);
        else if (left > 0) store_edge<XT>(p, v, int(left));
      }
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

}  // namespace rq
