// Matrix product of two MXFP4 operands: y = xq W^T + bias, xq the rows of x quantized as a
// weight is (mx4_codec.hip), in 4 bits all the way to gfx950's scaled matrix instructions:
// v_mfma_scale_f32_32x32x64_f8f6f4 takes 32 codes and their scale a lane and operand, which
// is one block, and sums in fp32.
//
// Tile BM x 256, 128 k a step, eight waves, two a SIMD.  Rows of 64 bytes of both operands
// come by direct-to-LDS loads into a ring of four steps, the four scales of a row and
// step as one dword likewise.  Lane (i, q) of part e of a step takes block 2 e + q of row i:
// 16 bytes, chunk c of row r stored at c ^ (r / 4) % 4, so that 16 consecutive rows' reads
// of a chunk meet no bank twice; the instruction picks byte 2 e of the row's scales,
// shifted by q bytes.  The operands of a part are read while the part before is multiplied.
// Products of many tiles run on the second kernel below.  4096 x 4096 x 14336: 143 us (3.4 PFLOP/s), 10 more for x's codes.
#include "rq_mx4_gemm.h"

namespace rq {
namespace {

constexpr int kA4Step = 128;

template <int BM_>
struct A4Tile {
  static constexpr int BM = BM_;
  static constexpr int WM = BM == 64 ? 1 : 2;
  static constexpr int WN = 8 / WM;
  static constexpr int MB = BM / (32 * WM);
  static constexpr int NB = 8 / WN;
  static constexpr int BN = 256;
  static constexpr int kRing = 4;
  static constexpr int kXBytes = BM * 64, kWBytes = BN * 64, kSBytes = 2048;
  static constexpr int kWOff = kXBytes, kSOff = kXBytes + kWBytes;
  static constexpr int kStage = kXBytes + kWBytes + kSBytes;
  static constexpr int kOutWave = mx_out_wave(MB, NB);
  static constexpr int kLds = kRing * kStage > 8 * kOutWave ? kRing * kStage : 8 * kOutWave;
  static constexpr int kXLoads = BM < 128 ? 1 : BM / 128;  // of a wave and step; BM = 64: half a wave's lanes
  static constexpr int kLoads = kXLoads + 2 + 1;
  static_assert(kLds <= 160 * 1024, "LDS plan");
};

struct A4Args {
  MxGemmArgs g;           // x: codes [M][pitch], codes, scales, wrows, pitch, cols, nk, splits, tiles, bias, y
  const uint8_t* xscales; // [M][xpitch / 16]
  int64_t xpitch;         // bytes of a row of x's codes
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ uint32_t swz64(uint32_t r, uint32_t c) { return r * 64u + ((c ^ ((r >> 2) & 3u)) << 4); }

// One direct-to-LDS load of 4 bytes a lane from an address of its own (see dma16).
__device__ __forceinline__ void dma4(const void* p, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(lds_addr) : "memory", "m0");
}

// 16 bytes a lane, likewise.
__device__ __forceinline__ void dma16_at(const void* p, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds_addr) : "memory", "m0");
}

// A wave-uniform value in scalar registers (the compiler may keep one that a masked load uses in vector registers).
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const uint8_t*>(uint64_t(uniform(uint32_t(v >> 32))) << 32 | uniform(uint32_t(v)));
}

// Rows m0 .. + count - 1, 256 columns from c0, nk steps from kbeg.
template <int XT, int BM, bool OUT32>
__device__ __forceinline__ void a4_tile(const A4Args& args, uint8_t* lds, int64_t m0, int count, int64_t c0, int split, int kbeg,
                                        int nk) {
  using T = A4Tile<BM>;
  constexpr int MB = T::MB, NB = T::NB, BN = T::BN;
  const MxGemmArgs& a = args.g;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  const int i32 = lane & 31, q = lane >> 5;

  // direct-to-LDS lanes: 16 rows an instruction; wave w brings the weight's rows 32 w .. and BM / 8 w .. of x
  const uint8_t* xbase = a.x + m0 * args.xpitch;
  const uint8_t* wbase = a.codes + c0 * a.pitch;
  const int wrows = a.wrows - c0 < BN ? int(a.wrows - c0) : BN;
  uint32_t xo[T::kXLoads], wo[2];
#pragma unroll
  for (int i = 0; i < T::kXLoads; ++i) {
    const int r = BM / 8 * wave + 16 * i + ((lane >> 2) & (BM == 64 ? 7 : 15));
    xo[i] = uint32_t(r < count ? r : count - 1) * uint32_t(args.xpitch) + 16u * (uint32_t(lane & 3) ^ ((r >> 2) & 3u));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * wave + 16 * i + (lane >> 2);
    wo[i] = uint32_t(r < wrows ? r : wrows - 1) * uint32_t(a.pitch) + 16u * (uint32_t(lane & 3) ^ ((r >> 2) & 3u));
  }
  // scales: lanes 0 .. 31 the weight's rows, the BM / 8 lanes after them x's
  const uint8_t* sp;
  {
    const int64_t srow = lane < 32 ? a.pitch / 16 : args.xpitch / 16;
    int r = lane < 32 ? 32 * wave + lane : BM / 8 * wave + ((lane - 32) & (BM / 8 - 1));
    const int most = lane < 32 ? wrows : count;
    r = r < most ? r : most - 1;
    sp = lane < 32 ? a.scales + (c0 + r) * srow : args.xscales + (m0 + r) * srow;
  }
  const uint32_t xdst = __builtin_amdgcn_readfirstlane(uint32_t(BM / 8 * wave) * 64u);
  const uint32_t wdst = __builtin_amdgcn_readfirstlane(uint32_t(wave) * 2048u);
  const uint32_t sdst = __builtin_amdgcn_readfirstlane(uint32_t(wave) * 256u);
  auto step_at = [&](int j) { return kbeg + (j < nk ? j : nk - 1); };  // past the end: the last step again, never used
  auto load_x = [&](int j) {
    const uint32_t st = uint32_t(j % T::kRing) * T::kStage;
    const int64_t k = int64_t(step_at(j)) * 64;
    if constexpr (BM == 64) {
      const uint8_t* p = uniform(xbase + k);
      const uint32_t to = uniform(st + xdst);
      if (lane < 32) dma16(p, xo[0], to);
    } else {
#pragma unroll
      for (int i = 0; i < T::kXLoads; ++i) dma16(uniform(xbase + k), xo[i], uniform(st + xdst + 1024u * i));
    }
  };
  auto load_w = [&](int j) {
    const uint32_t st = uint32_t(j % T::kRing) * T::kStage;
    const int kk = step_at(j);
    const int64_t k = int64_t(kk) * 64;
#pragma unroll
    for (int i = 0; i < 2; ++i) dma16(uniform(wbase + k), wo[i], uniform(st + T::kWOff + wdst + 1024u * i));
    const uint32_t to = uniform(st + T::kSOff + sdst);
    if (lane < 32 + BM / 8) dma4(sp + int64_t(kk) * 4, to);
  };

  f32x16 acc[MB][NB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[mb][nb][r] = 0.0f;

  const uint32_t xrow = uint32_t(32 * MB * wm + i32), wrow = uint32_t(32 * NB * wn + i32);
  u32x4 xf[2][MB], wf[2][NB];
  uint32_t xs[MB], ws[NB];
  auto read = [&](int buf, int j, int e) {
    const uint8_t* st = lds + uint32_t(j % T::kRing) * T::kStage;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      wf[buf][nb] = *reinterpret_cast<const u32x4*>(st + T::kWOff + swz64(wrow + 32 * nb, uint32_t(2 * e + q)));
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
      xf[buf][mb] = *reinterpret_cast<const u32x4*>(st + swz64(xrow + 32 * mb, uint32_t(2 * e + q)));
  };
  auto read_s = [&](int j) {
    const uint8_t* st = lds + uint32_t(j % T::kRing) * T::kStage + T::kSOff;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t r = wrow + 32 * nb;
      ws[nb] = *reinterpret_cast<const uint32_t*>(st + (r >> 5) * 256 + (r & 31) * 4) >> (8 * q);
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const uint32_t r = xrow + 32 * mb;
      xs[mb] = *reinterpret_cast<const uint32_t*>(st + r / (BM / 8) * 256 + 128 + r % (BM / 8) * 4) >> (8 * q);
    }
  };
  auto widen = [](const u32x4& v) { return i32x8{int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0}; };

#define RQ_A4_PRODUCTS(BUF, N0, N1, BYTE)                                                                                      \
  _Pragma("unroll") for (int nb = N0; nb < N1; ++nb)                                                                           \
  _Pragma("unroll") for (int mb = 0; mb < MB; ++mb)                                                                            \
    acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(wf[BUF][nb]), widen(xf[BUF][mb]), acc[mb][nb], 4, 4,   \
                                                                  BYTE, int(ws[nb]), BYTE, int(xs[mb]))
  load_x(0), load_w(0);
  load_x(1), load_w(1);
  load_x(2), load_w(2);
  step_barrier<2 * T::kLoads>();
  read(0, 0, 0);
  read_s(0);
  for (int j = 0; j < nk; ++j) {
    // the loads of step j + 3 are issued between products (together after the barrier they kept all waves
    // from their first product while the addresses went out)
    step_barrier<T::kLoads>();
    read(1, j, 1);
    __builtin_amdgcn_sched_barrier(0);
    RQ_A4_PRODUCTS(0, 0, 1, 0);
    __builtin_amdgcn_sched_barrier(0);
    load_x(j + 3);
    __builtin_amdgcn_sched_barrier(0);
    RQ_A4_PRODUCTS(0, 1, NB, 0);
    __builtin_amdgcn_sched_barrier(0);
    load_w(j + 3);
    read(0, j + 1, 0);
    __builtin_amdgcn_sched_barrier(0);
    RQ_A4_PRODUCTS(1, 0, NB, 2);
    __builtin_amdgcn_sched_barrier(0);
    read_s(j + 1);
  }
#undef RQ_A4_PRODUCTS
  wait_vmcnt<0>();
  __syncthreads();
  mx_output<XT, false, MB, NB, OUT32>(a, acc, lds + wave * T::kOutWave, lane, 0, true, split, m0, count, 32 * MB * wm,
                                      c0 + 32 * NB * wn);
}

// Tile t of n in order: an XCD (workgroup % 8) takes a run of tiles.
__device__ __forceinline__ int a4_run(int t, int n) { return t < n / 8 * 8 ? (t & 7) * (n / 8) + (t >> 3) : t; }

// Row and column tile of tile t: groups of four row tiles walked column by column.
__device__ __forceinline__ void a4_place(const MxGemmArgs& a, int t, int& rt, int& ct) {
  constexpr int GM = 4;
  const int per = GM * a.col_tiles, grp = t / per, r = t - grp * per;
  const int gm = a.row_tiles - grp * GM < GM ? a.row_tiles - grp * GM : GM;
  rt = grp * GM + r % gm;
  ct = r / gm;
}

template <int XT, int BM, bool OUT32>
__global__ __launch_bounds__(kMgThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mx4_a4_kernel(A4Args args) {
  const MxGemmArgs& a = args.g;
  __shared__ __attribute__((aligned(16))) uint8_t lds[A4Tile<BM>::kLds];
  lds_escapes(lds);
  int rt, ct;
  a4_place(a, a4_run(blockIdx.x, a.row_tiles * a.col_tiles), rt, ct);
  const int64_t m0 = int64_t(BM) * rt;
  const int split = blockIdx.y;
  const int kbeg = int(int64_t(a.nk) * split / a.splits), nk = int(int64_t(a.nk) * (split + 1) / a.splits) - kbeg;
  a4_tile<XT, BM, OUT32>(args, lds, m0, a.rows.M - m0 < BM ? int(a.rows.M - m0) : BM, int64_t(256) * ct, split, kbeg, nk);
}

// ---------------------------------------------------------------------------
// Many rows: 256 x 256 tiles, 256 k a step.  A cache line of a row's codes is 256 k, and what bounds the kernel above
// with many tiles is the number of lines it asks the L2 for (half a line of codes, and one more for
// four bytes of scales, a row and step: 0.73 requests a channel and cycle, the matrix units busy 36 %); here a step
// takes whole lines, and 16 bytes of a row's scales are asked for every second step.
//
// Wave (wr, wc) = (wave / 4, wave % 4) owns rows 64 wr .. + 63 and columns 32 wc .. + 31 of each 128 x 128
// quadrant, two blocks of 32 x 32.  A phase is a quadrant's eight products (256 cycles) behind the phase's
// LDS reads and one half tile's loads (128 rows, 16 KiB); waves 4 - 7 run one phase slot behind waves 0 - 3, so
// that of the two waves of a SIMD one reads while the other multiplies.  A half tile is refilled in the phase after its
// last reads, two steps ahead of its next use, and the waits leave the youngest six in flight.
//
// No unit is near its limit: 4096 x 8192 x 8192 at 3.7 PFLOP/s reads 1.7 GB from the L2 in 138 us (12.4 of the 33 TB/s that reads
// alone reach), the matrix units busy 49 to 55 % (4096 x 4096 x 14336: 15.5 TB/s and 41 %, LDS 25 %); waves wait for 39 % of
// their cycles (there are eight barriers a step; which of the waits it is was not resolved).  Power takes the clock from 2.4 to
// 1.9 GHz (8192 x 8192 x 8192 291 us, on zeros 230).  Four waves of 128 x 128 outputs, which read two thirds as much from LDS,
// took the same time to 3 %, and bringing lines to the L2 four steps ahead took 6 % more.
// ---------------------------------------------------------------------------
constexpr int kBgHalf = 128 * 128;                    // bytes of a half tile
constexpr int kBgStep = 4 * kBgHalf;                  // X0 X1 W0 W1
constexpr int kBgScales = 512 * 16;                   // two steps' scales: 256 rows of x, then the weight's
constexpr int kBgSOff = 2 * kBgStep;
constexpr int kBgRing = kBgSOff + 3 * kBgScales;
constexpr int kBgPitch = 256 * 2 + 16;                // the staged output tile's rows
constexpr int kBgLds = kBgRing > 256 * kBgPitch ? kBgRing : 256 * kBgPitch;
static_assert(kBgLds <= 160 * 1024 && A4Tile<128>::kLds <= kBgLds, "LDS plan");

template <int XT>
__global__ __launch_bounds__(kMgThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mx4_a4_big_kernel(A4Args args) {
  const MxGemmArgs& a = args.g;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kBgLds];
  lds_escapes(lds);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 2, wc = wave & 3;
  const int i32 = lane & 31, q = lane >> 5;
  int rt, ct;
  {
    // Tiles past the last whole round of compute units run as halves of their rows where these take one round, by the
    // kernel above's steps (896 tiles of 4096 x 4096 x 14336: 146 -> 143 us).
    const int G = a.row_tiles * a.col_tiles, rest = 2 * (G % a.cus) <= a.cus ? G % a.cus : 0, t = blockIdx.x;
    if (t >= G - rest) {
      const int v = a4_run(t - (G - rest), 2 * rest);
      a4_place(a, G - rest + (v >> 1), rt, ct);
      const int64_t m0 = int64_t(256) * rt + 128 * (v & 1);
      const int count = a.rows.M - m0 < 128 ? int(a.rows.M - m0) : 128;
      if (count > 0) a4_tile<XT, 128, false>(args, lds, m0, count, int64_t(256) * ct, 0, 0, int(a.pitch / 64));
      return;
    }
    a4_place(a, a4_run(t, G - rest), rt, ct);
  }
  const int64_t m0 = int64_t(256) * rt, c0 = int64_t(256) * ct;
  const int xrows = a.rows.M - m0 < 256 ? int(a.rows.M - m0) : 256;
  const int wrows = a.wrows - c0 < 256 ? int(a.wrows - c0) : 256;
  const int nk = a.nk;  // steps; the weight's last may be half of one (x has zeros there)

  // direct-to-LDS lanes: half tile h: rows 128 h + 16 wave + 8 i + lane / 8, chunk swizzled.  Where the weight's last
  // step is half of one, its second half's chunks are the first's again and their scales 2^-127.
  const uint8_t* xbase = a.x + m0 * args.xpitch;
  const uint8_t* wbase = a.codes + c0 * a.pitch;
  uint32_t xo[2][2], wo[2][2], back[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * wave + 8 * i + (lane >> 3);
    const uint32_t c = uint32_t(lane & 7) ^ ((r >> 1) & 7);
    back[i] = c >= 4 ? 64u : 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int rx = 128 * h + r < xrows ? 128 * h + r : xrows - 1, rw = 128 * h + r < wrows ? 128 * h + r : wrows - 1;
      xo[h][i] = uint32_t(rx) * uint32_t(args.xpitch) + 16u * c;
      wo[h][i] = uint32_t(rw) * uint32_t(a.pitch) + 16u * c;
    }
  }
  const bool half = a.pitch % 128 != 0;
  const uint32_t dst0 = __builtin_amdgcn_readfirstlane(uint32_t(wave) * 2048u);
  auto load_x = [&](int h, int step, uint32_t at) {
    const uint8_t* p = xbase + int64_t(step < nk ? step : nk - 1) * 128;  // past the end: the last step again, never used
    dma16(p, xo[h][0], dst0 + at);
    dma16(p, xo[h][1], dst0 + at + 1024u);
  };
  auto load_w = [&](int h, int step, uint32_t at) {
    const int st = step < nk ? step : nk - 1;
    const uint8_t* p = wbase + int64_t(st) * 128;
    const bool cut = half && st == nk - 1;
    dma16(p, wo[h][0] - (cut ? back[0] : 0u), dst0 + at);
    dma16(p, wo[h][1] - (cut ? back[1] : 0u), dst0 + at + 1024u);
  };
  // scales of steps 2 g, 2 g + 1: 16 bytes of row (tid) of x or of the weight; near a row's end its last 16 bytes
  const int xrow = int(args.xpitch / 16), wrow = int(a.pitch / 16);
  const uint8_t* sbase;
  {
    const int r = tid & 255, most = tid < 256 ? xrows : wrows;
    const int rr = r < most ? r : most - 1;
    sbase = tid < 256 ? args.xscales + (m0 + rr) * xrow : a.scales + (c0 + rr) * wrow;
  }
  auto group_at = [](int g, int row) { return 16 * g < row - 16 ? 16 * g : row - 16; };
  auto load_scales = [&](int g) {
    const int last = (nk - 1) / 2, gg = g < last ? g : last;
    const uint32_t to = __builtin_amdgcn_readfirstlane(uint32_t(kBgSOff + g % 3 * kBgScales) + 1024u * uint32_t(wave));
    dma16_at(sbase + (wave < 4 ? group_at(gg, xrow) : group_at(gg, wrow)), to);
  };
  auto xoff = [](int b, int h) { return uint32_t(b * kBgStep + h * kBgHalf); };
  auto woff = [](int b, int h) { return uint32_t(b * kBgStep + (2 + h) * kBgHalf); };
  // operand reads: chunk 2 s + q of the lane's row is its block of product s
  uint32_t xr[4], wrd[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    xr[s] = swz(uint32_t(64 * wr + i32), uint32_t(2 * s + q));
    wrd[s] = swz(uint32_t(32 * wc + i32), uint32_t(2 * s + q));
  }
  f32x16 acc[2][2][2];  // quadrant (hm, hn), block mb
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i >> 2][(i >> 1) & 1][i & 1][r] = 0.0f;
  u32x4 xa[2][4], w[2][4];
  uint32_t xs[2][2], ws[2][2];  // scales of a row: products 0 and 1 in bytes 0 and 2 of the first, 2 and 3 of the second
  // a step's scales: in its group's buffer, at the step's place in the row's 16 bytes
  const uint32_t sx = uint32_t(kBgSOff + 16 * (64 * wr + i32)), sw = uint32_t(kBgSOff + 16 * (256 + 32 * wc + i32));
  auto read_x = [&](int t, int b, int h) {
    const uint32_t at = sx + uint32_t(t / 2 % 3 * kBgScales + 8 * t - group_at(t / 2, xrow));
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
#pragma unroll
      for (int s = 0; s < 4; ++s) xa[mb][s] = *reinterpret_cast<const u32x4*>(lds + xoff(b, h) + mb * 4096 + xr[s]);
#pragma unroll
      for (int d = 0; d < 2; ++d) xs[mb][d] = *reinterpret_cast<const uint32_t*>(lds + at + 16 * (128 * h + 32 * mb) + 4 * d) >> (8 * q);
    }
  };
  auto read_w = [&](u32x4 (&o)[4], uint32_t (&so)[2], int step, int b, int h) {
    const int t = step < nk ? step : nk - 1;
    const uint32_t at = sw + uint32_t(t / 2 % 3 * kBgScales + 8 * t - group_at(t / 2, wrow));
#pragma unroll
    for (int s = 0; s < 4; ++s) o[s] = *reinterpret_cast<const u32x4*>(lds + woff(b, h) + wrd[s]);
#pragma unroll
    for (int d = 0; d < 2; ++d) so[d] = *reinterpret_cast<const uint32_t*>(lds + at + 16 * 128 * h + 4 * d) >> (8 * q);
    if (half && t == nk - 1) so[1] = 0;
  };
  auto widen = [](const u32x4& v) { return i32x8{int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0}; };
#define RQ_BG_MEM_END()                                                                 \
  do {                                                                                  \
    __builtin_amdgcn_sched_barrier(0);                                                  \
    asm volatile("s_waitcnt vmcnt(12) lgkmcnt(0)\n\ts_barrier" ::: "memory");          \
    __builtin_amdgcn_sched_barrier(0);                                                  \
  } while (0)
#define RQ_BG_MMA_END()                          \
  do {                                           \
    __builtin_amdgcn_sched_barrier(0);           \
    asm volatile("s_barrier" ::: "memory");      \
    __builtin_amdgcn_sched_barrier(0);           \
  } while (0)
#define RQ_BG_MMA1(C, W, WS, S)                                                                                             \
  _Pragma("unroll") for (int mb = 0; mb < 2; ++mb) C[mb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(                  \
      widen(W[S]), widen(xa[mb][S]), C[mb], 4, 4, (S & 1) * 2, int(WS[S / 2]), (S & 1) * 2, int(xs[mb][S / 2]))
#define RQ_BG_MMA(C, W, WS)         \
  do {                              \
    __builtin_amdgcn_s_setprio(1);  \
    RQ_BG_MMA1(C, W, WS, 0);        \
    RQ_BG_MMA1(C, W, WS, 1);        \
    RQ_BG_MMA1(C, W, WS, 2);        \
    RQ_BG_MMA1(C, W, WS, 3);        \
    __builtin_amdgcn_s_setprio(0);  \
  } while (0)
  // step t in buffer F = t % 2, which is also the weight half it starts with, so that a step's first can be read
  // while the step before multiplies by its other
#define RQ_BG_STEP(t, F)                                             \
  do {                                                               \
    read_x(t, F, 0);                                                 \
    load_w(F, (t) + 2, woff(F, F));                                  \
    if ((F) == 0) load_scales((t) / 2 + 2);                          \
    RQ_BG_MEM_END();                                                 \
    RQ_BG_MMA(acc[0][F], w[F], ws[F]);                               \
    RQ_BG_MMA_END();                                                 \
    read_w(w[1 - (F)], ws[1 - (F)], t, F, 1 - (F));                  \
    load_x(0, (t) + 2, xoff(F, 0));                                  \
    RQ_BG_MEM_END();                                                 \
    RQ_BG_MMA(acc[0][1 - (F)], w[1 - (F)], ws[1 - (F)]);             \
    RQ_BG_MMA_END();                                                 \
    read_x(t, F, 1);                                                 \
    load_w(1 - (F), (t) + 2, woff(F, 1 - (F)));                      \
    RQ_BG_MEM_END();                                                 \
    RQ_BG_MMA(acc[1][1 - (F)], w[1 - (F)], ws[1 - (F)]);             \
    RQ_BG_MMA_END();                                                 \
    read_w(w[1 - (F)], ws[1 - (F)], (t) + 1, 1 - (F), 1 - (F));      \
    load_x(1, (t) + 2, xoff(F, 1));                                  \
    RQ_BG_MEM_END();                                                 \
    RQ_BG_MMA(acc[1][F], w[F], ws[F]);                               \
    RQ_BG_MMA_END();                                                 \
  } while (0)
  load_scales(0);
  load_scales(1);
  load_w(0, 0, woff(0, 0));
  load_x(0, 0, xoff(0, 0));
  load_w(1, 0, woff(0, 1));
  load_x(1, 0, xoff(0, 1));
  load_w(1, 1, woff(1, 1));
  load_x(0, 1, xoff(1, 0));
  load_w(0, 1, woff(1, 0));
  load_x(1, 1, xoff(1, 1));
  RQ_BG_MEM_END();
  read_w(w[0], ws[0], 0, 0, 0);
  RQ_BG_MEM_END();
  if (wr == 1) RQ_BG_MMA_END();  // waves 4 - 7 run one slot behind
  int t = 0;
  for (; t + 2 <= nk; t += 2) {
    RQ_BG_STEP(t, 0);
    RQ_BG_STEP(t + 1, 1);
  }
  if (t < nk) RQ_BG_STEP(t, 0);
  if (wr == 0) asm volatile("s_barrier" ::: "memory");
  step_barrier<0>();
#undef RQ_BG_STEP
#undef RQ_BG_MMA
#undef RQ_BG_MMA1
#undef RQ_BG_MMA_END
#undef RQ_BG_MEM_END

  // Output: lane (i32, q) holds row i32 of a block, columns 8 h + 4 q .. + 3 in registers 4 h ..; the tile is
  // staged in LDS and stored 512 bytes a row.
  const int64_t left = a.cols - c0 < 256 ? a.cols - c0 : 256;
  const __amdgpu_buffer_rsrc_t br =
      buffer_rsrc(static_cast<const uint8_t*>(a.bias) + (a.bias ? c0 * 2 : 0), a.bias ? uint32_t(left * 2) : 0u);
#pragma unroll
  for (int hn = 0; hn < 2; ++hn)
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int col = 128 * hn + 32 * wc + 8 * h + 4 * q;
      float bias[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) bias[c] = from_x16<XT>(buf_load2(br, 2u * uint32_t(col + c)));
#pragma unroll
      for (int hm = 0; hm < 2; ++hm)
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          float v[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = __fadd_rn(acc[hm][hn][mb][4 * h + c], bias[c]);
          *reinterpret_cast<u32x2*>(lds + (128 * hm + 64 * wr + 32 * mb + i32) * kBgPitch + 2 * col) =
              u32x2{cvt_pk<XT>(v[0], v[1]), cvt_pk<XT>(v[2], v[3])};
        }
    }
  __syncthreads();
#pragma unroll 4
  for (int it = 0; it < 16; ++it) {
    const int r = 32 * wave + 2 * it + (lane >> 5);
    if (r >= xrows) continue;
    const u32x4 v = *reinterpret_cast<const u32x4*>(lds + r * kBgPitch + 16 * (lane & 31));
    const int64_t col = c0 + 8 * (lane & 31);
    uint16_t* p = static_cast<uint16_t*>(a.y) + (m0 + r) * a.ldy + col;
    if (col + 8 <= a.cols) store16_any(p, v);
    else if (col < a.cols) store_edge<XT>(p, v, int(a.cols - col));
  }
}

struct A4Plan {
  int bm, splits;
  bool big;
  int64_t xp;  // values of a row of x's codes
  int row_tiles, col_tiles;
  int64_t ld, codes_bytes, scales_bytes, part_bytes;
};

A4Plan a4_plan(const MxCall& c, int cus) {
  A4Plan p{};
  const int64_t wp = mx_pad(c.wk);
  p.bm = c.M <= 64 ? 64 : c.M <= 128 ? 128 : 256;
  p.col_tiles = int(ceil_div(c.N, 256));
  while (p.bm > 128 && 2 * ceil_div(c.M, p.bm) * p.col_tiles <= cus) p.bm /= 2;
  p.row_tiles = int(ceil_div(c.M, p.bm));
  const int64_t steps = wp / kA4Step;
  int64_t s = cus / (int64_t(p.row_tiles) * p.col_tiles);
  s = s < steps / 4 ? s : steps / 4;
  s = s < 16 ? s : 16;
  p.splits = int(s > 1 ? s : 1);
  p.big = p.bm == 256 && p.splits == 1 && c.dt != RQ_DTYPE_F32 && wp >= 512;
  p.ld = (c.N + 3) / 4 * 4;
  p.xp = p.big ? ceil_div(wp, 256) * 256 : wp;
  p.codes_bytes = up256(c.M * p.xp / 2);
  p.scales_bytes = up256(c.M * p.xp / kMxBlock);
  p.part_bytes = p.splits > 1 ? up256(int64_t(p.splits) * c.M * p.ld * 4) : 0;
  return p;
}

template <int XT, int BM>
void a4_launch(const A4Args& a, bool out32, hipStream_t stream) {
  const dim3 grid(unsigned(a.g.row_tiles) * unsigned(a.g.col_tiles), unsigned(a.g.splits));
  if (out32) mx4_a4_kernel<RQ_DTYPE_BF16, BM, true><<<grid, kMgThreads, 0, stream>>>(a);
  else mx4_a4_kernel<XT, BM, false><<<grid, kMgThreads, 0, stream>>>(a);
}

template <int XT>
void a4_launch_bm(const A4Args& a, int bm, bool out32, hipStream_t stream) {
  if (bm == 64) a4_launch<XT, 64>(a, out32, stream);
  else if (bm == 128) a4_launch<XT, 128>(a, out32, stream);
  else a4_launch<XT, 256>(a, out32, stream);
}

}  // namespace

int64_t mx4_a4_scratch(const MxCall& c, int cus) {
  const A4Plan p = a4_plan(c, cus);
  return p.codes_bytes + p.scales_bytes + p.part_bytes;
}

void mx4_a4_tiles(const MxCall& c, int cus, int32_t* out) {
  const A4Plan p = a4_plan(c, cus);
  out[0] = p.bm;
  out[1] = p.splits;
  out[2] = 1;
}

int mx4_a4_run(const MxCall& c, int cus) {
  const A4Plan p = a4_plan(c, cus);
  if (int64_t(p.row_tiles) * p.col_tiles > (int64_t(1) << 22)) return RQ_ERR_UNSUPPORTED;
  const int64_t wp = mx_pad(c.wk);
  uint8_t* xc = static_cast<uint8_t*>(c.scratch);
  uint8_t* xs = xc + p.codes_bytes;
  const int st = mx4_quantize(c.x, c.dt, c.M, c.K, c.ldx, xc, xs, p.xp, c.stream);
  if (st != RQ_OK) return st;
  A4Args a{};
  a.xpitch = p.xp / 2;
  a.xscales = xs;
  a.g.x = xc;
  a.g.rows = c.rows;
  a.g.codes = c.codes;
  a.g.scales = c.scales;
  a.g.wrows = a.g.cols = c.N;
  a.g.pitch = wp / 2;
  a.g.nk = int(wp / kA4Step);
  a.g.splits = p.splits;
  a.g.row_tiles = p.row_tiles;
  a.g.col_tiles = p.col_tiles;
  a.g.bias = c.bias;
  a.g.bias_dt = c.dt;
  const bool partial = p.splits > 1;
  void* part = xs + p.scales_bytes;
  a.g.y = partial ? part : c.y;
  a.g.ldy = partial ? p.ld : c.ldy;
  const bool out32 = partial || c.dt == RQ_DTYPE_F32;
  if (p.big) {
    a.g.nk = int(ceil_div(wp, 256));
    a.g.cus = cus;
    const int tiles = p.row_tiles * p.col_tiles, rest = tiles % cus;
    const unsigned grid = unsigned(tiles + (2 * rest <= cus ? rest : 0));
    if (c.dt == RQ_DTYPE_F16) mx4_a4_big_kernel<RQ_DTYPE_F16><<<grid, kMgThreads, 0, c.stream>>>(a);
    else mx4_a4_big_kernel<RQ_DTYPE_BF16><<<grid, kMgThreads, 0, c.stream>>>(a);
    return rq_check_launch();
  }
  if (c.dt == RQ_DTYPE_F16) a4_launch_bm<RQ_DTYPE_F16>(a, p.bm, out32, c.stream);
  else a4_launch_bm<RQ_DTYPE_BF16>(a, p.bm, out32, c.stream);
  if (partial) mx4_sum(MxSumArgs{static_cast<const float*>(part), c.M, p.ld, p.splits, 1, c.M, c.N, c.y, c.ldy}, c.dt, c.stream);
  return rq_check_launch();
}

}  // namespace rq
