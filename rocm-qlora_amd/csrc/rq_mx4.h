// MXFP4 (OCP microscaling): 32 consecutive values of a row share a power of two,
// each is an e2m1 code (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign).  With m = max |x|
// of a block,
//   e = floor(log2 m) - 2, clamped to -127 .. 127;  code = RNE_e2m1(x 2^-e), |.| <= 6.
// The stored scale byte is e + 127 (255: the block holds an infinity or a NaN and
// stands for NaN).  A value has two significant bits, so code 2^e is exact in bf16
// and fp32, and in fp16 for e = -23 .. 13 (rounded, or an infinity, outside).
//
// Rows are held in whole 128 values (zero codes after the last): codes are rows of
// Kp / 2 bytes, two a byte with the even value in the low bits, scales rows of Kp /
// 32 bytes, Kp = K rounded up to 128.  So a row's codes are 16-byte aligned and its
// scales 4-byte aligned, and a kernel's steps of 64 or 128 values have no remainder.
#pragma once

#include "rq_io.h"
#include "rq_launch.h"
#include "rq_rows.h"

namespace rq {

constexpr int kMxBlock = 32;
constexpr int kMxWhole = 128;

__host__ __device__ constexpr int64_t mx_pad(int64_t K) { return (K + kMxWhole - 1) / kMxWhole * kMxWhole; }

// Whether all of `rows` rows of `pitch` 16-bit values lie within 32-bit offsets of the first, read 128 bytes a step.
__host__ __device__ constexpr bool mx_rows_reached(int64_t rows, int64_t pitch) {
  return (rows - 1) * pitch * 2 + 128 <= int64_t(1) << 32;
}

// Scale byte of a block whose largest |x| has the fp32 bits `absmax` (an exponent field
// of 0 is a zero or below 2^-126: the least scale).
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t absmax) {
  const int f = int(absmax >> 23);
  return f == 255 ? 255u : uint32_t(f > 2 ? f - 2 : 0);
}

// The scale as the conversion instructions take it: an fp32 number's exponent field (0 is
// 2^-127 to them, 255 a NaN).
__device__ __forceinline__ float mx_scale(uint32_t byte) { return u2f(byte << 23); }

// Byte B of `word`, two codes, as a pair of 16-bit values.
template <int XT, int B>
__device__ __forceinline__ uint32_t mx_pair(uint32_t word, float scale) {
  if constexpr (XT == RQ_DTYPE_F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, B));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, B));
}

// Eight codes as eight 16-bit values.
template <int XT>
__device__ __forceinline__ u32x4 mx_decode8(uint32_t word, float scale) {
  return u32x4{mx_pair<XT, 0>(word, scale), mx_pair<XT, 1>(word, scale), mx_pair<XT, 2>(word, scale),
               mx_pair<XT, 3>(word, scale)};
}

// fp32 x = hi + mid + lo in bf16, exactly but for what lies below 2^-133: eight bits by
// truncation each time, so that no part overflows.  An infinity or a NaN is hi alone (a NaN
// whose payload truncation would clear is set quiet).
struct Split3 {
  uint32_t hi, mid, lo;  // bf16 bits in the upper half
};
__device__ __forceinline__ Split3 mx_split(float x) {
  const uint32_t b = f2u(x);
  if ((b & 0x7F800000u) == 0x7F800000u) return Split3{(b & 0x7FFFFFu) ? (b | 0x400000u) & 0xFFFF0000u : b, 0u, 0u};
  const uint32_t h = b & 0xFFFF0000u;
  const float r = __fsub_rn(x, u2f(h));
  const uint32_t m = f2u(r) & 0xFFFF0000u;
  const uint32_t l = f2u(__fsub_rn(r, u2f(m))) & 0xFFFF0000u;
  return Split3{h, m, l};
}

// ---- the linears' arguments, as the entry points check them ------------------------
// y[r] = x[r / xdiv] W[e(r)]^T + bias[e(r)], e(r) the row's expert in `rows` (a null plan:
// expert 0); rows without an expert are zeros.  dX: the same with W for W^T.
struct MxCall {
  const void* x;
  int dt;
  int64_t M, K, ldx;  // rows of the product, x's columns
  bool aligned16;     // x's rows are 16-byte aligned
  int xdiv;           // product rows that read one row of x
  RowsPlan rows;
  const uint8_t* codes;   // [E][N][Kp / 2]
  const uint8_t* scales;  // [E][N][Kp / 32]
  int64_t E, N, wk;       // the weight's rows and (unpadded) columns
  const void* bias;       // [E][out columns] of dt, or null
  void* y;
  int64_t ldy;
  int ysum;               // dX: rows of the product that one row of y is the sum of
  bool dx, a4;
  void* scratch;
  hipStream_t stream;
};

inline int64_t up256(int64_t n) { return (n + 255) & ~int64_t(255); }

// `pitch`: values of a row of codes, whole 128.
int mx4_quantize(const void* x, int dt, int64_t rows, int64_t cols, int64_t ld, uint8_t* codes, uint8_t* scales, int64_t pitch,
                 hipStream_t stream);
// A copy of rows, zeros up to `pitch` values (a multiple of 8).
void mx4_rows_whole(const void* x, int dt, int64_t rows, int64_t cols, int64_t ld, void* out, int64_t pitch, hipStream_t stream);
// The kernel for few rows (mx4_few.hip): x's rows in whole steps take at most kMxFewBytes.
constexpr uint32_t kMxFewBytes = 0xFFFFFFE0u;  // (kOobOffset is past them)
int64_t mx4_few_scratch(const MxCall& c);
int mx4_few_run(const MxCall& c);
int mx4_gemm_run(const MxCall& c, int cus);
int64_t mx4_gemm_scratch(const MxCall& c, int cus);
int mx4_a4_run(const MxCall& c, int cus);
int64_t mx4_a4_scratch(const MxCall& c, int cus);
// Rows of a tile, splits of the contraction, whether the rows are copied (or quantized) first.
void mx4_gemm_tiles(const MxCall& c, int cus, int32_t* out);
void mx4_a4_tiles(const MxCall& c, int cus, int32_t* out);

}  // namespace rq
