// The 8-bit activation checkpoint's codec (rq_act8.h).
//
// Bound by memory: a value is read once and 33/32 of a byte written (and back).
// A thread takes 16 values, two threads a block, so that codes leave as whole
// 16-byte stores and the block's maximum is one lane swap.  4096 x 14336 bf16 (178 MB a way):
// 29 us to codes and 28 back, 6.1 and 6.4 TB/s (a copy reaches 5.2; part of the codes stays in
// the cache between the two); 333 x 1001 3 us each, a launch.
#include "rq_act8.h"
#include "rq_io.h"
#include "rq_launch.h"

namespace rq {
namespace {

constexpr int kA8Threads = 256;
constexpr int kA8Vals = 16;  // values of a thread

struct Act8Args {
  int64_t rows, cols;
  int64_t ld;        // of the values
  int64_t pitch;     // of the codes: cols rounded up to 32
  int64_t groups;    // pitch / 16
};

// This thread's row and first column.
__device__ __forceinline__ void act8_place(const Act8Args& a, int64_t& row, int64_t& col) {
  const int64_t b0 = int64_t(blockIdx.x) * kA8Threads;
  const int64_t r0 = b0 / a.groups;  // uniform
  const uint64_t at = uint64_t(b0 - r0 * a.groups) + threadIdx.x;
  if (uint64_t(a.groups) + kA8Threads <= 0xFFFFFFFFu) {
    const uint32_t q = uint32_t(at) / uint32_t(a.groups);
    row = r0 + q;
    col = int64_t(uint32_t(at) - q * uint32_t(a.groups)) * kA8Vals;
  } else {
    row = r0 + int64_t(at / uint64_t(a.groups));
    col = int64_t(at % uint64_t(a.groups)) * kA8Vals;
  }
}

template <int XT>
__global__ __launch_bounds__(kA8Threads) void act8_quantize_kernel(Act8Args a, const void* x, uint8_t* codes,
                                                                   uint8_t* exps) {
  constexpr int V = Elem<XT>::kVec;
  int64_t row, col;
  act8_place(a, row, col);
  const bool live = row < a.rows;  // both threads of a block alike: a row's groups are even in number
  float v[kA8Vals];
  const typename Elem<XT>::T* p = static_cast<const typename Elem<XT>::T*>(x) + (live ? row * a.ld + col : 0);
  u32x4 raw[kA8Vals / V];
  if (live && col + kA8Vals <= a.cols) {
#pragma unroll
    for (int i = 0; i < kA8Vals / V; ++i) raw[i] = load16_any(p + V * i);
  } else {
#pragma unroll
    for (int i = 0; i < kA8Vals / V; ++i) raw[i] = load16_part<XT>(p + V * i, live ? a.cols - col - V * i : 0);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kA8Vals / V; ++i) {
    float f[V];
    unpack16<XT>(raw[i], f);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[V * i + e] = f[e];
      // the bits of |x| order as the values do, with NaN on top
      const uint32_t m = f2u(f[e]) & 0x7FFFFFFFu;
      top = m > top ? m : top;
    }
  }
  const uint32_t other = __shfl_xor(top, 1);
  top = other > top ? other : top;
  if (!live) return;
  const int e = act8_exponent(top);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = act8_code(v[4 * i + k], e);
    // bytes 0 of c0..c3
    w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0C0C0400u),
                                 __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u), 0x05040100u);
    if (e == kAct8NoScale) w[i] = 0u;
  }
  *reinterpret_cast<u32x4*>(codes + row * a.pitch + col) = u32x4{w[0], w[1], w[2], w[3]};
  if ((col & 16) == 0) exps[row * (a.pitch / kAct8Block) + col / kAct8Block] = uint8_t(e);
}

template <int XT>
__global__ __launch_bounds__(kA8Threads) void act8_dequantize_kernel(Act8Args a, const uint8_t* codes,
                                                                     const uint8_t* exps, void* out) {
  constexpr int V = Elem<XT>::kVec;
  int64_t row, col;
  act8_place(a, row, col);
  if (row >= a.rows) return;
  const u32x4 w = *reinterpret_cast<const u32x4*>(codes + row * a.pitch + col);
  const int e = exps[row * (a.pitch / kAct8Block) + col / kAct8Block];
  float v[kA8Vals];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[4 * i] = act8_value<0>(w[i], e);
    v[4 * i + 1] = act8_value<1>(w[i], e);
    v[4 * i + 2] = act8_value<2>(w[i], e);
    v[4 * i + 3] = act8_value<3>(w[i], e);
  }
  typename Elem<XT>::T* p = static_cast<typename Elem<XT>::T*>(out) + row * a.ld + col;
#pragma unroll
  for (int i = 0; i < kA8Vals / V; ++i) {
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = v[V * i + k];
    store16_part<XT>(p + V * i, f, a.cols - col - V * i);
  }
}

// Rows that lie end to end and fill whole blocks are one long row.
int act8_args(int64_t rows, int64_t cols, int64_t ld, Act8Args* a, int64_t* blocks) {
  if (rows < 0 || cols < 1 || ld < cols || cols > (int64_t(1) << 40) || rows > (int64_t(1) << 40)) return RQ_ERR_BAD_SHAPE;
  if (rows > 0 && cols > (int64_t(1) << 40) / rows) return RQ_ERR_UNSUPPORTED;
  a->rows = rows;
  a->cols = cols;
  a->ld = ld;
  if (cols % kAct8Block == 0 && ld == cols && rows > 1) {
    a->cols = a->ld = rows * cols;
    a->rows = 1;
  }
  a->pitch = ceil_div(a->cols, kAct8Block) * kAct8Block;
  a->groups = a->pitch / kA8Vals;
  *blocks = ceil_div(a->rows * a->groups, kA8Threads);
  return *blocks > kMaxThreads1D / kA8Threads ? RQ_ERR_UNSUPPORTED : RQ_OK;
}

}  // namespace
}  // namespace rq

extern "C" int rq_act8_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes,
                                uint8_t* exponents, hipStream_t stream) {
  using namespace rq;
  if (!valid_float_dtype(x_dtype)) return RQ_ERR_BAD_DTYPE;
  Act8Args a{};
  int64_t blocks = 0;
  const int st = act8_args(rows, cols, ldx, &a, &blocks);
  if (st != RQ_OK || rows == 0) return st;
  if (!x || !codes || !exponents) return RQ_ERR_NULL_POINTER;
  if (!aligned(x, dtype_size(x_dtype)) || !aligned(codes, 16)) return RQ_ERR_BAD_ALIGNMENT;
  RQ_DISPATCH_DT(x_dtype, XT, act8_quantize_kernel<XT><<<unsigned(blocks), kA8Threads, 0, stream>>>(a, x, codes, exponents));
  return rq_check_launch();
}

extern "C" int rq_act8_dequantize(const uint8_t* codes, const uint8_t* exponents, int64_t rows, int64_t cols, void* out,
                                  int out_dtype, int64_t ldo, hipStream_t stream) {
  using namespace rq;
  if (!valid_float_dtype(out_dtype)) return RQ_ERR_BAD_DTYPE;
  Act8Args a{};
  int64_t blocks = 0;
  const int st = act8_args(rows, cols, ldo, &a, &blocks);
  if (st != RQ_OK || rows == 0) return st;
  if (!codes || !exponents || !out) return RQ_ERR_NULL_POINTER;
  if (!aligned(out, dtype_size(out_dtype)) || !aligned(codes, 16)) return RQ_ERR_BAD_ALIGNMENT;
  RQ_DISPATCH_DT(out_dtype, XT, act8_dequantize_kernel<XT><<<unsigned(blocks), kA8Threads, 0, stream>>>(a, codes, exponents, out));
  return rq_check_launch();
}
