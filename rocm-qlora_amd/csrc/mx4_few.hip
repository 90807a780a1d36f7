// Few rows beside an MXFP4 weight (decoding): y = x W^T + bias, rows grouped by expert
// or all of one weight.
//
// A workgroup takes 16 NB rows of the weight and a tile of at most 64 rows of x (rq_rows.h), its eight waves
// two adjacent steps of 128 k of every sixteen each.  Lane (i, g) = (l % 16, l / 16) loads block g of a step of
// weight row i, 16 bytes; the 4 x 4 dwords of four lane groups are turned by four lane swaps, so that operand s of
// v_mfma_f32_16x16x32 is k = 32 s + 8 g .. and a wave reads x in whole 64-byte pieces of its rows (in the order of
// the blocks each 16-byte piece was a line of its own: 16 rows beside 14336 x 4096 took 26 us).  A batch of steps'
// loads, x's among them, are issued before its first product; a weight is read and decoded once for all rows of a
// pass.  The waves' sums meet in LDS and are added in wave order, 16 rows of x to a wave.
//
// Bound by memory latency and by x, which every workgroup reads from the L2: 4096 -> 4096 with 1, 16 and 32 bf16 rows
// 5.5, 8.1 and 12.9 us (1.6 TB/s of weight with 1), 4096 -> 14336 with 16 rows 12.8 us (2.4 TB/s), 64 experts'
// 4096 -> 2048 with 64 rows 47 us (3.7 TB/s).
//
// fp32 rows: x = hi + mid + lo in bf16 (exact, rq_mx4.h), three products a value, all
// into the same fp32 sum.  Activations in 4 bits: x's codes and scales instead of values,
// one v_mfma_scale_f32_16x16x128_f8f6f4 a step, nothing decoded.
#include "rq_mx4.h"

namespace rq {
namespace {

constexpr int kFwWaves = 8;
constexpr int kFwThreads = 64 * kFwWaves;

struct FewArgs {
  const void* x;           // rows 16-byte aligned, within 32-bit offsets
  const uint8_t* xscales;  // 4 bits: [rows][wp / 32]
  uint32_t xsbytes;        // of them all: the last row's last step may be the first of a load of two
  int64_t ldx;             // elements (4 bits: bytes)
  int64_t wp;              // columns of x and of the weight, whole steps
  int xdiv;
  RowsPlan rows;
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t N;
  const void* bias;
  void* y;
  int64_t ldy;
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

// dword d of lane group g <-> dword g of lane group d
__device__ __forceinline__ void turn4(u32x4& v) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  u2 p = __builtin_amdgcn_permlane32_swap(v.x, v.z, false, false);
  u2 r = __builtin_amdgcn_permlane32_swap(v.y, v.w, false, false);
  u2 a = __builtin_amdgcn_permlane16_swap(p.x, r.x, false, false);
  u2 b = __builtin_amdgcn_permlane16_swap(p.y, r.y, false, false);
  v = u32x4{a.x, a.y, b.x, b.y};
}

// Steps of a batch, as registers allow.  One chunk of rows: a wave's whole share of a contraction of 4096
// or, for 16 columns, 8192 is asked for at once (each batch waits for memory: 1.5 to 2 us).  More
// chunks: two batches are in flight, rows of all chunks among them.
constexpr int few_depth(bool a4, bool f32, int ch, int nb, bool deep) {
  int d = ch == 1 ? (deep ? 8 : 4) : nb == 1 ? (a4 && ch == 2 ? 4 : 2) : nb == 2 ? 2 : 1;
  return f32 && d > 1 ? d / 2 : d;
}

// XT: x's and y's dtype.  A4: activations in 4 bits.  CH: chunks of 16 rows of x in one pass.
// DEEP: longer batches (one chunk of rows, NB = 1).
template <int XT, bool A4, int CH, int NB, bool DEEP>
__global__ __launch_bounds__(kFwThreads) __attribute__((amdgpu_waves_per_eu(2)))
void mx4_few_kernel(FewArgs a) {
  typedef typename Elem<XT>::T T;
  constexpr int ES = int(sizeof(T));
  constexpr int OT = XT == RQ_DTYPE_F16 ? RQ_DTYPE_F16 : RQ_DTYPE_BF16;  // operand type
  constexpr int V = Elem<XT>::kVec, P = A4 ? 1 : 8 / V;  // pieces of 16 bytes of an operand
  constexpr int D = few_depth(A4, XT == RQ_DTYPE_F32, CH, NB, DEEP);
  constexpr int kX = A4 ? 1 : 4 * P;  // 16-byte pieces of x of a lane and step
  __shared__ f32x4 red[kFwWaves][CH][NB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  const int i = lane & 15, g = lane >> 4;
  // An expert's rows of the first pass, asked for beside the tile (of slots not in use: anything).  Not with NB = 4, whose
  // 127 registers let two workgroups share a compute unit (64 experts' 2048 columns of 4096 beside 64 rows: 47 us, with
  // registers for one 55).
  constexpr bool kEarly = CH == 1 && NB < 4;
  const int first = kEarly ? plan_row(a.rows, int64_t(kTileRows) * blockIdx.y + i) : 0;
  const Tile tile = plan_tile(a.rows, blockIdx.y);
  if (tile.count == 0) return;
  const int64_t n0 = int64_t(blockIdx.x) * (16 * NB);
  const int64_t expert = __builtin_amdgcn_readfirstlane(tile.adapter < 0 ? 0 : tile.adapter);
  const int64_t slot0 = int64_t(kTileRows) * blockIdx.y;
  const int steps = __builtin_amdgcn_readfirstlane(tile.adapter < 0 ? 0 : int(a.wp / kMxWhole));

  // Loads go by buffers without a branch around them: a lane without a row, a row past the last and a step
  // past the last read zeros at an offset out of bounds, and the waits count what is in flight.
  const int64_t left = a.N - n0 < 16 * NB ? a.N - n0 : 16 * NB;
  const uint32_t pitch = uint32_t(a.wp / 2), spitch = uint32_t(a.wp / kMxBlock);
  const __amdgpu_buffer_rsrc_t wr = buffer_rsrc(a.codes + (expert * a.N + n0) * pitch, uint32_t(left) * pitch);
  const __amdgpu_buffer_rsrc_t sr = buffer_rsrc(a.scales + (expert * a.N + n0) * spitch, uint32_t(left) * spitch);
  const __amdgpu_buffer_rsrc_t xr = buffer_rsrc(a.x, kMxFewBytes), xsr = buffer_rsrc(A4 ? a.xscales : a.scales, A4 ? a.xsbytes : 0u);
  // a wave's steps: two adjacent ones of every sixteen
  const int batches = (2 * ((steps + 15) / 16) + D - 1) / D;
  auto step_of = [&](int b, int d) { return 16 * ((b * D + d) / 2) + 2 * wave + ((b * D + d) & 1); };
  struct W {
    u32x4 c[D][NB];
    uint32_t s[D][NB];
  };
  auto load_w = [&](W& w, int b) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int st = step_of(b, d);
      const uint32_t off = uint32_t(i) * pitch + 16u * g + 64u * uint32_t(st);
      const uint32_t soff = uint32_t(i) * spitch + 4u * uint32_t(st);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        w.c[d][nb] = buf_load16(wr, st < steps ? off + 16u * nb * pitch : kOobOffset);
        const uint32_t at = st < steps ? soff + 16u * nb * spitch : kOobOffset;
        if constexpr (D == 1) {
          w.s[d][nb] = buf_load4(sr, at);
        } else if (d % 2 == 0) {  // two steps' (a 4-byte load of 16 rows costs as much as a 16-byte one)
          const u32x2 two = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(sr, at, 0, 0));
          w.s[d][nb] = two.x;
          w.s[d + 1][nb] = st + 1 < steps ? two.y : 0u;  // (not another row's: 255 times a code of zero is a NaN)
        }
      }
    }
  };
  uint32_t bias[NB][4];  // as loaded; without one zeros
  {
    const bool on = a.bias && tile.adapter >= 0;
    const __amdgpu_buffer_rsrc_t br =
        buffer_rsrc(static_cast<const uint8_t*>(a.bias) + (on ? (expert * a.N + n0) * ES : 0), on ? uint32_t(left) * ES : 0u);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t off = uint32_t(ES) * (16 * nb + 4 * g + r);
        if constexpr (XT == RQ_DTYPE_F32) bias[nb][r] = buf_load4(br, off);
        else bias[nb][r] = buf_load2(br, off);
      }
  }

  // 16 CH rows of the tile at a time (one pass, but for an expert with more than its share)
  for (int at0 = 0; at0 < tile.count; at0 += 16 * CH) {
    int row[CH];       // this lane's row of x in each chunk
    uint32_t xo[CH];   // its offset
    uint32_t xso[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int at = at0 + 16 * c + i;
      row[c] = at < tile.count ? (kEarly && at0 == 0 ? first : plan_row(a.rows, slot0 + at)) : -1;
      const uint32_t r = uint32_t(row[c] < 0 ? 0 : row[c]) / uint32_t(a.xdiv);
      xo[c] = r * uint32_t(a.ldx * (A4 ? 1 : ES)) + (A4 ? 16u * g : uint32_t(8 * ES) * g);
      xso[c] = A4 ? r * spitch : 0u;
    }
    struct X {
      u32x4 v[D][kX];
      uint32_t s[D];
    };
    // operand s of step d in pieces P s ..; past a row's end zeros
    auto load_x = [&](X& x, int b, int c) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int st = step_of(b, d);
        const bool on = row[c] >= 0 && st < steps;
        if constexpr (A4) {
          x.v[d][0] = buf_load16(xr, on ? xo[c] + 64u * uint32_t(st) : kOobOffset);
          const uint32_t at = on ? xso[c] + 4u * uint32_t(st) : kOobOffset;
          if constexpr (D == 1) {
            x.s[d] = buf_load4(xsr, at);
          } else if (d % 2 == 0) {
            const u32x2 two = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(xsr, at, 0, 0));
            x.s[d] = two.x;
            x.s[d + 1] = st + 1 < steps ? two.y : 0u;
          }
        } else {
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j < P; ++j) {
              x.v[d][P * s + j] = buf_load16(xr, on ? xo[c] + uint32_t(ES) * (128u * uint32_t(st) + 32u * s + V * j) : kOobOffset);
            }
        }
      }
    };
    f32x4 acc[CH][NB];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) acc[c][nb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto products = [&](int c, const u32x4 (&wv)[NB][A4 ? 1 : 4], const uint32_t (&wsc)[NB], const u32x4 (&x)[kX], uint32_t xsc) {
      if constexpr (A4) {
        const i32x8 xa = {int(x[0].x), int(x[0].y), int(x[0].z), int(x[0].w), 0, 0, 0, 0};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const u32x4& v = wv[nb][0];
          const i32x8 wa = {int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0};
          acc[c][nb] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xa, acc[c][nb], 4, 4, 0, int(wsc[nb] >> (8 * g)), 0,
                                                                       int(xsc >> (8 * g)));
        }
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if constexpr (XT == RQ_DTYPE_F32) {
            u32x4 h, m, l;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const u32x4& v = x[2 * s + (j >> 1)];
              const Split3 e = mx_split(u2f(v[2 * (j & 1)])), o = mx_split(u2f(v[2 * (j & 1) + 1]));
              h[j] = e.hi >> 16 | o.hi;
              m[j] = e.mid >> 16 | o.mid;
              l[j] = e.lo >> 16 | o.lo;
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              acc[c][nb] = mfma16x16x32<OT>(wv[nb][s], l, acc[c][nb]);
              acc[c][nb] = mfma16x16x32<OT>(wv[nb][s], m, acc[c][nb]);
              acc[c][nb] = mfma16x16x32<OT>(wv[nb][s], h, acc[c][nb]);
            }
          } else {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) acc[c][nb] = mfma16x16x32<OT>(wv[nb][s], x[s], acc[c][nb]);
          }
        }
      }
    };
    auto decode = [&](W& w, int d, u32x4 (&wv)[NB][A4 ? 1 : 4]) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if constexpr (A4) {
          wv[nb][0] = w.c[d][nb];
        } else {
          turn4(w.c[d][nb]);
#pragma unroll
          for (int s = 0; s < 4; ++s) wv[nb][s] = mx_decode8<OT>(w.c[d][nb][s], mx_scale(w.s[d][nb] >> (8 * s) & 255u));
        }
      }
    };

    if constexpr (CH == 1) {
      for (int b = 0; b < batches; ++b) {
        W w;
        X x;
        load_w(w, b);
        load_x(x, b, 0);
#pragma unroll
        for (int d = 0; d < D; ++d) {
          u32x4 wv[NB][A4 ? 1 : 4];
          decode(w, d, wv);
          products(0, wv, w.s[d], x.v[d], x.s[d]);
        }
      }
    } else {
      // a batch: the next one's weight and rows are asked for, then this one's are multiplied
      W wb[2];
      X xb[2][CH];
      auto load = [&](W& w, X (&x)[CH], int b) {
        load_w(w, b);
#pragma unroll
        for (int c = 0; c < CH; ++c) load_x(x[c], b, c);
      };
      auto batch = [&](W& w, X (&x)[CH]) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
          u32x4 wv[NB][A4 ? 1 : 4];  // for all chunks
          decode(w, d, wv);
#pragma unroll
          for (int c = 0; c < CH; ++c) products(c, wv, w.s[d], x[c].v[d], x[c].s[d]);
        }
      };
      load(wb[0], xb[0], 0);
      for (int b = 0; b + 2 <= batches; b += 2) {
        load(wb[1], xb[1], b + 1);
        batch(wb[0], xb[0]);
        load(wb[0], xb[0], b + 2);
        batch(wb[1], xb[1]);
      }
      if (batches & 1) batch(wb[0], xb[0]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) red[wave][c][nb][lane] = acc[c][nb];
    __syncthreads();
    // chunk c and block nb to wave (c + CH nb) % 8; lane (i, g): row of x i, columns 4 g .. + 3
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if ((c + CH * nb) % kFwWaves != wave || row[c] < 0) continue;
        f32x4 sum = red[0][c][nb][lane];
#pragma unroll
        for (int w = 1; w < kFwWaves; ++w) {
          const f32x4 v = red[w][c][nb][lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[r] = __fadd_rn(sum[r], v[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (XT == RQ_DTYPE_F32) sum[r] = __fadd_rn(sum[r], u2f(bias[nb][r]));
          else sum[r] = __fadd_rn(sum[r], from_x16<XT>(bias[nb][r]));
        }
        const int64_t no = n0 + 16 * nb + 4 * g;
        T* yp = static_cast<T*>(a.y) + int64_t(row[c]) * a.ldy + no;
        if (no + 4 <= a.N) {
          if constexpr (XT == RQ_DTYPE_F32) store16_any(yp, u32x4{f2u(sum[0]), f2u(sum[1]), f2u(sum[2]), f2u(sum[3])});
          else *reinterpret_cast<u32x2_any*>(yp) = u32x2_any{cvt_pk<XT>(sum[0], sum[1]), cvt_pk<XT>(sum[2], sum[3])};
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (no + r < a.N) yp[r] = from_f32<XT>(sum[r]);
        }
      }
    __syncthreads();
  }
}

template <int XT, bool A4, int CH, int NB>
void few_launch(const FewArgs& a, hipStream_t stream) {
  const dim3 grid(unsigned(ceil_div(a.N, 16 * NB)), unsigned(a.rows.T));
  if (CH == 1 && NB == 1 && a.wp > 4096) mx4_few_kernel<XT, A4, CH, NB, CH == 1 && NB == 1><<<grid, kFwThreads, 0, stream>>>(a);
  else mx4_few_kernel<XT, A4, CH, NB, false><<<grid, kFwThreads, 0, stream>>>(a);
}

template <int XT, bool A4, int CH>
void few_launch(const FewArgs& a, int nb, hipStream_t stream) {
  if (nb == 1) few_launch<XT, A4, CH, 1>(a, stream);
  else if (nb == 2) few_launch<XT, A4, CH, 2>(a, stream);
  else few_launch<XT, A4, CH, 4>(a, stream);
}

template <int XT, bool A4>
int few_launch(const FewArgs& a, hipStream_t stream) {
  // Blocks of a workgroup: as many as still leave a workgroup or so for each compute unit (14336 columns beside
  // 16 rows: 25, 18 and 16 us with 1, 2 and 4; 4096 columns: 9, 11 and 14; 16 experts' 1024 columns of 2048 - 10 us with 2, 11
  // with 4 - and 32's 13 and 15; their 2048 of 4096 21 and 20).
  const bool grouped = a.rows.p != nullptr;
  const int64_t blocks = ceil_div(a.N, 16) * a.rows.T;
  const int nb = blocks > (grouped ? 1024 : 768) ? 4 : blocks > 384 ? 2 : 1;
  // Chunks of a pass: all of one weight's rows (fp32 rows: at most 16 come here).  An expert has few rows: a chunk, and a
  // pass more where it has more (64 experts' 2048 columns of 4096 beside 64 rows: 47 us, with two chunks a pass 66).
  if constexpr (XT != RQ_DTYPE_F32 || A4) {
    if (!grouped && a.rows.M > 32 && A4) {
      few_launch<XT, A4, A4 ? 4 : 1>(a, nb, stream);
      return rq_check_launch();
    }
    if (!grouped && a.rows.M > 16) {
      few_launch<XT, A4, 2>(a, nb, stream);
      return rq_check_launch();
    }
  }
  few_launch<XT, A4, 1>(a, nb, stream);
  return rq_check_launch();
}

}  // namespace

// Codes of x, or a copy of rows that the kernel does not read as they are.
static bool few_copies(const MxCall& c) {
  return !c.aligned16 || c.K != mx_pad(c.wk) || ceil_div(c.M, c.xdiv) * c.ldx * int64_t(dtype_size(c.dt)) > int64_t(kMxFewBytes);
}

int64_t mx4_few_scratch(const MxCall& c) {
  const int64_t rows = ceil_div(c.M, c.xdiv), wp = mx_pad(c.wk);
  if (c.a4) return up256(rows * wp / 2) + up256(rows * wp / kMxBlock);
  return few_copies(c) ? up256(rows * wp * int64_t(dtype_size(c.dt))) : 0;
}

int mx4_few_run(const MxCall& c) {
  FewArgs a{};
  const int64_t rows = ceil_div(c.M, c.xdiv);
  a.x = c.x;
  a.ldx = c.ldx;
  a.wp = mx_pad(c.wk);
  a.xdiv = c.xdiv;
  a.rows = c.rows;
  a.codes = c.codes;
  a.scales = c.scales;
  a.N = c.N;
  a.bias = c.bias;
  a.y = c.y;
  a.ldy = c.ldy;
  if (c.a4) {
    uint8_t* xc = static_cast<uint8_t*>(c.scratch);
    uint8_t* xs = xc + up256(rows * a.wp / 2);
    const int st = mx4_quantize(c.x, c.dt, rows, c.K, c.ldx, xc, xs, a.wp, c.stream);
    if (st != RQ_OK) return st;
    a.x = xc;
    a.ldx = a.wp / 2;
    a.xscales = xs;
    a.xsbytes = uint32_t(rows * (a.wp / kMxBlock));
    RQ_DISPATCH_DT(c.dt, XT, return few_launch<XT, true>(a, c.stream));
  }
  if (few_copies(c)) {
    mx4_rows_whole(c.x, c.dt, rows, c.K, c.ldx, c.scratch, a.wp, c.stream);
    a.x = c.scratch;
    a.ldx = a.wp;
  }
  RQ_DISPATCH_DT(c.dt, XT, return few_launch<XT, false>(a, c.stream));
  return RQ_OK;
}

}  // namespace rq
