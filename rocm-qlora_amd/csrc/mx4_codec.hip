// MXFP4 codec (format: rq_mx4.h).  Both directions are bound by memory: four lanes
// share a block, a lane holds 8 values of it (16 bytes of 16-bit values, one
// instruction's 1 KiB a wave), the block's largest |x| is found by lane swaps, and
// gfx950's own conversions, which take the power of two with them, round and pack.
// 14336 x 4096 in bf16: 25.4 us to codes (5.9 TB/s), 22.7 back (6.5 TB/s; part of the codes still in the cache).
#include "rq_mx4.h"

namespace rq {
namespace {

constexpr int kMxThreads = 256;
constexpr int kMxVals = 8;  // values of a lane and group
constexpr int kMxDepth = 4; // groups of a lane, loaded before the first is used

struct MxCodecArgs {
  int64_t rows, cols, ld;
  int64_t groups;  // groups of 8 values of a padded row
};

// fp32 bits of the largest |value| of 16 or 32 bytes (any NaN is above any number).
template <int XT>
__device__ __forceinline__ uint32_t absmax_bits(const u32x4 (&v)[XT == RQ_DTYPE_F32 ? 2 : 1]) {
  uint32_t m = 0;
  if constexpr (XT == RQ_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) m = max(m, v[i][k] & 0x7FFFFFFFu);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) m = max(m, max((v[0][k] << 16) & 0x7FFF0000u, v[0][k] & 0x7FFF0000u));
    if constexpr (XT == RQ_DTYPE_F16) m = f2u(f16_to_f32(uint16_t(m >> 16)));
  }
  return m;
}

template <int XT>
__device__ __forceinline__ uint32_t encode8(const u32x4 (&v)[XT == RQ_DTYPE_F32 ? 2 : 1], float s) {
  uint32_t q = 0;
  const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};  // (a bit cast of a vector's element takes its first)
  if constexpr (XT == RQ_DTYPE_F32) {
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, u2f(v[0][0]), u2f(v[0][1]), s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, u2f(v[0][2]), u2f(v[0][3]), s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, u2f(v[1][0]), u2f(v[1][1]), s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, u2f(v[1][2]), u2f(v[1][3]), s, 3);
  } else if constexpr (XT == RQ_DTYPE_BF16) {
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[0]), s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[1]), s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[2]), s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[3]), s, 3);
  } else {
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[0]), s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[1]), s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[2]), s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[3]), s, 3);
  }
  return q;
}

// The largest of four adjacent lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), 0xB1, 0xF, 0xF, true)));  // lanes 1 0 3 2
  return max(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), 0x4E, 0xF, 0xF, true)));  // lanes 2 3 0 1
}

// Group g of a workgroup's lane and depth d: adjacent lanes take adjacent groups.
__device__ __forceinline__ int64_t codec_group(int d) {
  return (int64_t(blockIdx.x) * kMxDepth + d) * blockDim.x + threadIdx.x;
}

template <int XT>
__global__ __launch_bounds__(kMxThreads) void mx4_quantize_kernel(MxCodecArgs a, const void* x, uint32_t* codes,
                                                                  uint8_t* scales) {
  typedef typename Elem<XT>::T T;
  constexpr int V = Elem<XT>::kVec, P = kMxVals / V;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const T* p = static_cast<const T*>(x) + row * a.ld;
    u32x4 v[kMxDepth][P];
#pragma unroll
    for (int d = 0; d < kMxDepth; ++d) {
      const int64_t c = codec_group(d) * kMxVals;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        v[d][i] = u32x4{0u, 0u, 0u, 0u};
        if (c + V * i < a.cols) v[d][i] = load16_part<XT>(p + c + V * i, a.cols - c - V * i);
      }
    }
#pragma unroll
    for (int d = 0; d < kMxDepth; ++d) {
      const int64_t g = codec_group(d);
      if (g >= a.groups) break;  // whole blocks: groups are a multiple of 16
      const uint32_t b = mx_scale_byte(quad_max(absmax_bits<XT>(v[d])));
      codes[row * a.groups + g] = b == 255u ? 0u : encode8<XT>(v[d], mx_scale(b));
      if ((g & 3) == 0) scales[row * (a.groups / 4) + g / 4] = uint8_t(b);
    }
  }
}

template <int XT>
__global__ __launch_bounds__(kMxThreads) void mx4_dequantize_kernel(MxCodecArgs a, const uint32_t* codes,
                                                                    const uint8_t* scales, void* out) {
  typedef typename Elem<XT>::T T;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    T* p = static_cast<T*>(out) + row * a.ld;
    uint32_t w[kMxDepth], b[kMxDepth];
#pragma unroll
    for (int d = 0; d < kMxDepth; ++d) {
      int64_t g = codec_group(d);
      g = g < a.groups ? g : a.groups - 1;
      w[d] = codes[row * a.groups + g];
      b[d] = scales[row * (a.groups / 4) + g / 4];
    }
#pragma unroll
    for (int d = 0; d < kMxDepth; ++d) {
      const int64_t c = codec_group(d) * kMxVals;
      if (c >= a.cols) break;
      const float s = mx_scale(b[d]);
      if constexpr (XT == RQ_DTYPE_F32) {
        float f[8];
        const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], s, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], s, 1);
        const f32x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], s, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[d], s, 3);
        const float lo[4] = {v0.x, v0.y, v1.x, v1.y}, hi[4] = {v2.x, v2.y, v3.x, v3.y};
        store16_part<XT>(p + c, lo, a.cols - c);
        if (c + 4 < a.cols) store16_part<XT>(p + c + 4, hi, a.cols - c - 4);
      } else {
        const u32x4 v = mx_decode8<XT>(w[d], s);
        if (c + 8 <= a.cols) store16_any(p + c, v);
        else store_edge<XT>(p + c, v, int(a.cols - c));
      }
    }
  }
}

// Rows that lie end to end and are whole are one long row.
int codec_args(int64_t rows, int64_t cols, int64_t ld, int64_t pitch, MxCodecArgs* a, dim3* grid, unsigned* threads) {
  if (rows < 0 || cols < 1 || ld < cols || cols > (int64_t(1) << 40) || rows > (int64_t(1) << 40)) return RQ_ERR_BAD_SHAPE;
  if (rows > 0 && cols > (int64_t(1) << 40) / rows) return RQ_ERR_UNSUPPORTED;
  *a = MxCodecArgs{rows, cols, ld, 0};
  a->groups = pitch / kMxVals;
  if (pitch == cols && ld == cols && rows > 1) {
    a->cols = a->ld = rows * cols;
    a->groups *= rows;
    a->rows = 1;
  }
  *threads = a->groups <= 64 * kMxDepth ? 64 : a->groups <= 128 * kMxDepth ? 128 : kMxThreads;
  const int64_t blocks = ceil_div(a->groups, int64_t(*threads) * kMxDepth);
  if (blocks * *threads > kMaxThreads1D) return RQ_ERR_UNSUPPORTED;
  *grid = dim3(unsigned(blocks), unsigned(a->rows < 32768 ? (a->rows > 0 ? a->rows : 1) : 32768));
  return RQ_OK;
}

}  // namespace

int mx4_quantize(const void* x, int dt, int64_t rows, int64_t cols, int64_t ld, uint8_t* codes, uint8_t* scales,
                 int64_t pitch, hipStream_t stream) {
  MxCodecArgs a{};
  dim3 grid;
  unsigned threads = 0;
  const int st = codec_args(rows, cols, ld, pitch, &a, &grid, &threads);
  if (st != RQ_OK || rows == 0) return st;
  RQ_DISPATCH_DT(dt, XT, mx4_quantize_kernel<XT><<<grid, threads, 0, stream>>>(a, x, reinterpret_cast<uint32_t*>(codes), scales));
  return rq_check_launch();
}

}  // namespace rq

extern "C" int rq_mx4_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes,
                               uint8_t* scales, hipStream_t stream) {
  using namespace rq;
  if (!valid_float_dtype(x_dtype)) return RQ_ERR_BAD_DTYPE;
  if (rows > 0 && (!x || !codes || !scales)) return RQ_ERR_NULL_POINTER;
  if (!aligned(x, dtype_size(x_dtype)) || !aligned(codes, 16)) return RQ_ERR_BAD_ALIGNMENT;
  return mx4_quantize(x, x_dtype, rows, cols, ldx, codes, scales, mx_pad(cols), stream);
}

extern "C" int rq_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* out,
                                 int out_dtype, int64_t ldo, hipStream_t stream) {
  using namespace rq;
  if (!valid_float_dtype(out_dtype)) return RQ_ERR_BAD_DTYPE;
  MxCodecArgs a{};
  dim3 grid;
  unsigned threads = 0;
  const int st = codec_args(rows, cols, ldo, mx_pad(cols), &a, &grid, &threads);
  if (st != RQ_OK || rows == 0) return st;
  if (!codes || !scales || !out) return RQ_ERR_NULL_POINTER;
  if (!aligned(out, dtype_size(out_dtype)) || !aligned(codes, 16)) return RQ_ERR_BAD_ALIGNMENT;
  RQ_DISPATCH_DT(out_dtype, XT, mx4_dequantize_kernel<XT><<<grid, threads, 0, stream>>>(
                                    a, reinterpret_cast<const uint32_t*>(codes), scales, out));
  return rq_check_launch();
}
