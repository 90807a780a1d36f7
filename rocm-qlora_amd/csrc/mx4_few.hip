// Few rows beside an MXFP4 weight (decoding): y = x W^T + bias, rows grouped by expert
// or all of one weight.
//
// A workgroup takes 16 rows of the weight and a tile of at most 64 rows of x (rq_rows.h),
// its eight waves every eighth step of 128 k.  Lane (i, g) = (l % 16, l / 16) holds block
// g of the step of weight row n0 + i: 16 bytes of codes, one scale, 32 values, which are
// four operands of v_mfma_f32_16x16x32 (the k order within a step is free as long as both
// operands have the same: operand s is values 8 s .. of each block).  x comes straight
// from memory in that order.  A weight is read and decoded once for all 64 rows.  The waves'
// sums meet in LDS and are added in wave order, 16 rows of x to a wave.
//
// fp32 rows: x = hi + mid + lo in bf16 (exact, rq_mx4.h), three products a value, all
// into the same fp32 sum.  Activations in 4 bits: x's codes and scales instead of values,
// one v_mfma_scale_f32_16x16x128_f8f6f4 a step, nothing decoded.
#include "rq_mx4.h"

namespace rq {
namespace {

constexpr int kFwWaves = 8;
constexpr int kFwThreads = 64 * kFwWaves;
constexpr int kFwCols = 16;   // weight rows of a workgroup
constexpr int kFwDepth = 4;   // steps of a wave in flight

struct FewArgs {
  const void* x;
  const uint8_t* xscales;  // 4 bits: [rows][wp / 32]
  int64_t ldx;             // elements (4 bits: bytes)
  int64_t K, wp;           // x's columns, the weight's padded ones
  int xdiv;
  bool vec;                // rows of x are 16-byte aligned and whole steps
  RowsPlan rows;
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t N;
  const void* bias;
  void* y;
  int64_t ldy;
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

// XT: x's and y's dtype.  A4: activations in 4 bits.  CH: chunks of 16 rows, at most.
template <int XT, bool A4, int CH>
__global__ __launch_bounds__(kFwThreads) void mx4_few_kernel(FewArgs a) {
  constexpr int OT = XT == RQ_DTYPE_F16 ? RQ_DTYPE_F16 : RQ_DTYPE_BF16;  // operand type
  __shared__ f32x4 red[kFwWaves][CH][64];
  const Tile tile = plan_tile(a.rows, blockIdx.y);
  if (tile.count == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int i = lane & 15, g = lane >> 4;
  const int64_t n0 = int64_t(blockIdx.x) * kFwCols;
  const int expert = tile.adapter < 0 ? 0 : tile.adapter;
  const int64_t slot0 = int64_t(kTileRows) * blockIdx.y;

  // this lane's row of x in each chunk (a live row where there is none: its result is not stored)
  int row[CH];
  const uint8_t* xp[CH];
  const uint8_t* xs[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int at = 16 * c + i;
    row[c] = at < tile.count ? plan_row(a.rows, slot0 + at) : -1;
    const int64_t r = (row[c] < 0 ? plan_row(a.rows, slot0) : row[c]) / a.xdiv;
    if constexpr (A4) {
      xp[c] = static_cast<const uint8_t*>(a.x) + r * a.ldx + 16 * g;
      xs[c] = a.xscales + r * (a.wp / kMxBlock) + g;
    } else {
      xp[c] = static_cast<const uint8_t*>(a.x) + r * a.ldx * int64_t(sizeof(typename Elem<XT>::T));
    }
  }
  f32x4 acc[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int steps = tile.adapter < 0 ? 0 : int(a.wp / kMxWhole);
  const int64_t n = n0 + i < a.N ? n0 + i : a.N - 1;  // past the last: a live row again, not stored
  const uint8_t* wc = a.codes + (int64_t(expert) * a.N + n) * (a.wp / 2) + 16 * g;
  const uint8_t* ws = a.scales + (int64_t(expert) * a.N + n) * (a.wp / kMxBlock) + g;
  for (int s0 = wave; s0 < steps; s0 += kFwWaves * kFwDepth) {
    u32x4 w[kFwDepth];
    uint32_t sc[kFwDepth];
#pragma unroll
    for (int d = 0; d < kFwDepth; ++d) {
      const int st = s0 + kFwWaves * d < steps ? s0 + kFwWaves * d : s0;
      w[d] = *reinterpret_cast<const u32x4*>(wc + int64_t(st) * 64);
      sc[d] = ws[int64_t(st) * 4];
    }
#pragma unroll
    for (int d = 0; d < kFwDepth; ++d) {
      const int st = s0 + kFwWaves * d;
      if (st >= steps) break;
      if constexpr (A4) {
        const i32x8 wa = {int(w[d].x), int(w[d].y), int(w[d].z), int(w[d].w), 0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          if (16 * c >= tile.count) break;
          const u32x4 v = *reinterpret_cast<const u32x4*>(xp[c] + int64_t(st) * 64);
          const i32x8 xa = {int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0};
          acc[c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xa, acc[c], 4, 4, 0, int(sc[d]), 0,
                                                                    int(xs[c][int64_t(st) * 4]));
        }
      } else {
        const float scale = mx_scale(sc[d]);
        u32x4 wv[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) wv[s] = mx_decode8<OT>(w[d][s], scale);
        const int64_t k = int64_t(st) * kMxWhole + 32 * g;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          if (16 * c >= tile.count) break;
          const typename Elem<XT>::T* p = reinterpret_cast<const typename Elem<XT>::T*>(xp[c]) + k;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            constexpr int V = Elem<XT>::kVec, P = 8 / V;
            u32x4 v[P];
#pragma unroll
            for (int j = 0; j < P; ++j) {
              const int64_t left = a.K - k - 8 * s - V * j;
              if (a.vec) v[j] = *reinterpret_cast<const u32x4*>(p + 8 * s + V * j);
              else v[j] = left > 0 ? load16_part<XT>(p + 8 * s + V * j, left) : u32x4{0u, 0u, 0u, 0u};
            }
            if constexpr (XT == RQ_DTYPE_F32) {
              u32x4 h, m, l;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const Split3 e = mx_split(u2f(v[j >> 1][2 * (j & 1)])), o = mx_split(u2f(v[j >> 1][2 * (j & 1) + 1]));
                h[j] = e.hi >> 16 | o.hi;
                m[j] = e.mid >> 16 | o.mid;
                l[j] = e.lo >> 16 | o.lo;
              }
              acc[c] = mfma16x16x32<OT>(wv[s], l, acc[c]);
              acc[c] = mfma16x16x32<OT>(wv[s], m, acc[c]);
              acc[c] = mfma16x16x32<OT>(wv[s], h, acc[c]);
            } else {
              acc[c] = mfma16x16x32<OT>(wv[s], v[0], acc[c]);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) red[wave][c][lane] = acc[c];
  __syncthreads();
  // wave c: chunk c; lane (i, g): row of x i, columns n0 + 4 g .. + 3
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (c != wave || row[c] < 0) continue;
    f32x4 sum = red[0][c][lane];
#pragma unroll
    for (int w = 1; w < kFwWaves; ++w)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum[r] = __fadd_rn(sum[r], red[w][c][lane][r]);
    typename Elem<XT>::T* yp = static_cast<typename Elem<XT>::T*>(a.y) + int64_t(row[c]) * a.ldy;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t no = n0 + 4 * g + r;
      if (no >= a.N) break;
      float v = sum[r];
      if (a.bias && tile.adapter >= 0) v = __fadd_rn(v, load_as_f32(a.bias, int64_t(expert) * a.N + no, XT));
      yp[no] = from_f32<XT>(v);
    }
  }
}

template <int XT, bool A4>
int few_launch(const FewArgs& a, int most, hipStream_t stream) {
  const dim3 grid(unsigned(ceil_div(a.N, kFwCols)), unsigned(a.rows.T));
  if (most <= 16) mx4_few_kernel<XT, A4, 1><<<grid, kFwThreads, 0, stream>>>(a);
  else if (most <= 32) mx4_few_kernel<XT, A4, 2><<<grid, kFwThreads, 0, stream>>>(a);
  else mx4_few_kernel<XT, A4, 4><<<grid, kFwThreads, 0, stream>>>(a);
  return rq_check_launch();
}

}  // namespace

int mx4_few_run(const MxCall& c) {
  FewArgs a{};
  const int es = int(dtype_size(c.dt));
  a.x = c.x;
  a.ldx = c.ldx;
  a.K = c.K;
  a.wp = mx_pad(c.wk);
  a.xdiv = c.xdiv;
  a.vec = c.K == a.wp && aligned(c.x, 16) && c.ldx * es % 16 == 0;
  a.rows = c.rows;
  a.codes = c.codes;
  a.scales = c.scales;
  a.N = c.N;
  a.bias = c.bias;
  a.y = c.y;
  a.ldy = c.ldy;
  const int most = int(c.M < kTileRows ? c.M : kTileRows);
  if (c.a4) {
    const int64_t rows = ceil_div(c.M, c.xdiv);
    uint8_t* xc = static_cast<uint8_t*>(c.scratch);
    uint8_t* xs = xc + rows * (a.wp / 2);
    const int st = mx4_quantize(c.x, c.dt, rows, c.K, c.ldx, xc, xs, c.stream);
    if (st != RQ_OK) return st;
    a.x = xc;
    a.ldx = a.wp / 2;
    a.xscales = xs;
    RQ_DISPATCH_DT(c.dt, XT, return few_launch<XT, true>(a, most, c.stream));
  }
  RQ_DISPATCH_DT(c.dt, XT, return few_launch<XT, false>(a, most, c.stream));
  return RQ_OK;
}

}  // namespace rq
