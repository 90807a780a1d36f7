// The 8-bit activation checkpoint: blocks of 32 consecutive values of a row
// share a power-of-two scale (the OCP MX format MXINT8).  With m = max |x| of a
// block,
//   E = floor(log2 m),  q = clamp(rne(x 2^(6 - E)), -127, 127),  x^ = q 2^(E - 6).
// The stored exponent byte is E + 127, which is the exponent field of m as an
// fp32 number (0 for zeros and subnormals: E = -127; 255 for an infinity or a
// NaN: the whole block stands for NaN).  q has 7 magnitude bits, so x^ is exact
// in bf16, fp16 (for blocks that fp16 values made) and fp32: what reads a
// checkpoint as a matrix operand rounds nothing.
//
// Codes are rows of ceil(cols / 32) * 32 bytes (zeros past cols), exponents rows
// of ceil(cols / 32) bytes.
#pragma once

#include "rq_common.h"
#include "rq_mfma.h"

namespace rq {

constexpr int kAct8Block = 32;
constexpr int kAct8NoScale = 255;

// Exponent byte of a block whose largest |x| has the fp32 bits `absmax`.
__device__ __forceinline__ int act8_exponent(uint32_t absmax) { return int(absmax >> 23); }

// The byte of q for x, in the low 8 bits (the others are not zero).  Adding
// 1.5 * 2^23 rounds to an integer, ties to even, and leaves its two's complement
// in the low bits.
__device__ __forceinline__ uint32_t act8_code(float x, int e) {
  const float v = __builtin_amdgcn_fmed3f(ldexpf(x, 6 + 127 - e), -127.0f, 127.0f);
  return f2u(__fadd_rn(v, 12582912.0f));
}

// 2^(E - 6) as ldexp's argument.
__device__ __forceinline__ int act8_shift(int e) { return e - 127 - 6; }

// x^ of byte B of `word`.
template <int B>
__device__ __forceinline__ float act8_value(uint32_t word, int e) {
  const float q = float(int32_t(word << (24 - 8 * B)) >> 24);
  return e == kAct8NoScale ? __builtin_nanf("") : ldexpf(q, act8_shift(e));
}

// Four codes as 16-bit operand pairs.
template <int XT>
__device__ __forceinline__ u32x2 act8_pairs(uint32_t word, int e) {
  return u32x2{cvt_pk<XT>(act8_value<0>(word, e), act8_value<1>(word, e)),
               cvt_pk<XT>(act8_value<2>(word, e), act8_value<3>(word, e))};
}

}  // namespace rq
