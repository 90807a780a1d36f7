// Matrix products of 16-bit rows and an MXFP4 weight for gfx950, one weight or one for
// each expert: y = x W^T + bias, and dX = dY W (the same kernel with the weight read the
// other way).
//
// The weight stays in 4 bits up to the registers.  gfx950 converts a byte of two codes and
// a scale to two bf16 (or fp16) values in one full-rate instruction; a wave of the 256 x 256
// tile issues 8 of them (dX: 16 and 16 byte permutes) beside 8 v_mfma_f32_32x32x16 of 32
// cycles each, and a second wave of the SIMD multiplies meanwhile: a loop of 8 products
// and 16 conversions takes the time of the products, with 16 permutes more 13 % longer.
// 4-bit tiles take a quarter of the LDS, of its reads and of the traffic to it.
//
// Tile BM x BN, 64 k a step, eight waves, two a SIMD; the weight is the products' A operand,
// so that a lane's results lie along an output row.  Rows come by direct-to-LDS loads into
// a ring of four steps (128-byte rows, swizzled; MgTile says where eight), codes likewise (dX: three); the loads
// of a step are issued two to three steps before its products, one barrier a step, and the operands of
// the next quarter step are read from LDS while this one's are multiplied.
//
// 4096 x 4096 x 14336 in bf16, replayed for seconds: forward 392 us (1.23 PFLOP/s), dX 411 (1.17); a library's products of the
// decoded weight 313 and 325, decoding it 23 more.  Bound by the loop's waits and by the clock: the matrix units are busy in 59 %
// of the cycles (dX 52, experts 54), LDS in 18 (20), the L2 gives 11.4 of the 33 TB/s that reads alone reach, and waves wait for
// 45 % of theirs (34); power takes the clock from 2.4 to 1.9 GHz (the same instructions on zeros: 312 us).  Experts: 2048 tokens'
// two of 8 of 4096 -> 14336 486 us (0.99 PFLOP/s of live rows: tiles' ends).
//
// Forward: lane (i, q) (i = l % 32, q = l / 32) of a 32-column block holds a whole block
// of 32 k of its weight row: one 16-byte LDS read and one scale a step; its quarter s
// are k = 32 q + 8 s .., and the rows' chunks are read in that order.  Scales come to registers, 8
// steps at a time.
//
// dX: the contraction runs over weight rows, the codes lie along columns.  Four adjacent codes are
// taken as one 16-bit element and ds_read_b64_tr_b16 turns 4 rows x 16 elements: lane i
// has columns 4 i .. 4 i + 3 of eight rows in four registers.  A conversion gives two columns of a row,
// a permute pairs the same column of two rows: operands of four blocks, block b holding
// columns 4 i + b, so that the four blocks' results of a lane are four adjacent outputs.  The
// scales, transposed and as bf16 once a call (1 / 16 of the codes), come by the same ring.
#include "rq_mx4_gemm.h"

namespace rq {
namespace {

// WM x WN waves of 32 MB x 32 NB outputs each.
//
// 64 rows.  Forward: a step's products of a wave take 256 cycles, so a barrier is passed every second step only
// and loads run six steps ahead (64 x 256 tiles, a step: 0.45 us with one step a barrier, three ahead).  dX: the two
// waves of a column block would decode the same weights for half the rows each; instead each takes all rows and
// half the quarters of every step (kShare), and they exchange half their sums at the end.
template <bool DX, int BM_>
struct MgTile {
  static constexpr int BM = BM_;
  static constexpr int kShare = DX && BM == 64 ? 2 : 1;  // waves that share a block's contraction
  static constexpr int WM = BM == 64 ? 1 : 2;
  static constexpr int WN = 8 / (WM * kShare);
  static constexpr int MB = BM / (32 * WM);
  static constexpr int NB = DX ? 4 : (BM == 64 ? 1 : 2);
  static constexpr int BN = 32 * NB * WN;
  static constexpr int kXBytes = BM * 128;
  static constexpr int kWRow = DX ? BN / 2 : 32;               // bytes of a tile row of codes
  static constexpr int kWBytes = DX ? kMgStep * kWRow : BN * kWRow;
  static constexpr int kSBytes = DX ? BN / 32 * 128 : 0;       // scales of a step
  static constexpr int kSteps = !DX && BM == 64 ? 2 : 1;       // steps a barrier (forward)
  static constexpr int kXRing = 4 * kSteps, kWRing = DX ? 3 : 4 * kSteps;
  static constexpr int kAhead = kXRing - kSteps;               // steps that a step's loads are ahead of it
  static constexpr int kWOff = kXRing * kXBytes;
  static constexpr int kSOff = kWOff + kWRing * kWBytes;
  static constexpr int kRing = kSOff + kWRing * kSBytes;
  static constexpr int kOutWave = mx_out_wave(MB / kShare, NB);
  static constexpr int kSwapWave = kShare == 2 ? 64 * 4 * 16 * NB : 0;  // bytes a wave hands to the one it shares with
  static constexpr int kEnd = 8 * (kOutWave > kSwapWave ? kOutWave : kSwapWave);
  static constexpr int kLds = kRing > kEnd ? kRing : kEnd;
  static constexpr int kXLoads = BM / 64, kWLoads = kWBytes / 8192;
  static constexpr int kLoads = kXLoads + kWLoads + (DX ? 1 : 0);  // of a wave and step
  static_assert(kLds <= 160 * 1024 && BN >= 256, "LDS plan");
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

// The rows of row tile rt: slots slot0 .. + count - 1 of one expert (-1: none).
struct MgRows {
  int expert, count;
  int64_t slot0;
};
template <int BM>
__device__ __forceinline__ MgRows mg_rows(const MxGemmArgs& a, int rt) {
  if (!a.rows.p) {
    const int64_t slot0 = int64_t(BM) * rt;
    return MgRows{0, a.rows.M - slot0 < BM ? int(a.rows.M - slot0) : BM, slot0};
  }
  int first = rt;  // 64-row tile
  if constexpr (BM > kTileRows) first = a.rows.p[a.rows.off_big() + (BM == 256 ? a.rows.bigs(0) : 0) + rt];
  const Tile tile = plan_tile(a.rows, first);
  int count = tile.count;
#pragma unroll
  for (int j = 1; j < BM / kTileRows; ++j) {
    if (first + j >= a.rows.T) break;
    const Tile next = plan_tile(a.rows, first + j);
    if (next.adapter != tile.adapter) break;
    count += next.count;
  }
  return MgRows{__builtin_amdgcn_readfirstlane(tile.adapter), __builtin_amdgcn_readfirstlane(count), int64_t(kTileRows) * first};
}

// One tile: rows R, columns of column tile ct.
template <int XT, bool DX, int BM, bool OUT32>
__device__ __forceinline__ void mg_tile(const MxGemmArgs& a, uint8_t* lds, const MgRows& R, int ct) {
  using T = MgTile<DX, BM>;
  constexpr int MB = T::MB, NB = T::NB, BN = T::BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = wave / (T::WM * T::WN);  // of a shared contraction
  const int wm = wave / T::WN % T::WM, wn = wave % T::WN;
  const int i32 = lane & 31, q = lane >> 5;
  const int expert = R.expert, count = R.count;
  const int64_t slot0 = R.slot0;
  const bool live = expert >= 0;  // rows without an expert are zeros
  const int64_t e = live ? expert : 0;
  const int64_t c0 = int64_t(BN) * ct;  // first output column

  const int all = a.planes * a.nk;
  // forward splits begin at even steps (a dword of scales is two steps)
  auto bound = [&](int s) { return DX ? int(int64_t(all) * s / a.splits) : 2 * int(int64_t(all / 2) * s / a.splits); };
  const int split = blockIdx.y;
  const int kbeg = bound(split);
  const int nk = live ? bound(split + 1) - kbeg : 0;

  f32x16 acc[MB][NB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[mb][nb][r] = 0.0f;

  if (nk > 0) {
    // direct-to-LDS lanes.  Rows: wave w brings rows BM / 8 w .. of the step, 8 an instruction;
    // 16-byte chunk c of row r is stored at chunk c ^ (r / 2) % 8.
    const uint8_t* xbase = a.x + (a.by_slot ? slot0 * a.ldx : 0);
    uint32_t xo[T::kXLoads];
#pragma unroll
    for (int i = 0; i < T::kXLoads; ++i) {
      const int r = BM / 8 * wave + 8 * i + (lane >> 3);
      const int rr = r < count ? r : count - 1;  // a live row again where there is none
      const uint32_t c = uint32_t(16 * ((lane & 7) ^ ((r >> 1) & 7)));
      const uint32_t row = a.by_slot ? uint32_t(rr) : uint32_t(plan_row(a.rows, slot0 + rr)) / uint32_t(a.xdiv);
      xo[i] = row * uint32_t(a.ldx) + c;  // (mg_plan takes no more rows than keep it under 4 GiB)
    }
    const uint32_t xdst = __builtin_amdgcn_readfirstlane(uint32_t(BM / 8 * wave) * 128u);
    // Codes.  Forward: rows of 32 bytes, wave w rows 32 w .. (+ 256 an instruction), chunk c of
    // row r at c ^ (r / 8) % 2.  dX: 64 rows of kWRow bytes, 32-byte piece p of row r at
    // p ^ f(r), which spreads the four rows of a transposing read over the banks.
    const uint8_t* wbase;
    uint32_t wo[T::kWLoads], wrow[T::kWLoads];
#pragma unroll
    for (int i = 0; i < T::kWLoads; ++i) {
      if constexpr (DX) {
        constexpr int kPer = T::kWRow / 16;  // chunks of a row
        const int at = 512 * i + tid, r = at / kPer, pos = at % kPer;
        const int f = kPer == 8 ? (r >> 1) & 3 : r & 7;
        const int64_t byte = c0 / 2 + 16 * (pos ^ (f << 1));
        wrow[i] = uint32_t(r);
        wo[i] = uint32_t(byte < a.pitch ? byte : a.pitch - 16);
      } else {
        const int r = 256 * i + 32 * wave + (lane >> 1);
        const int64_t n = c0 + r < a.wrows ? c0 + r : a.wrows - 1;
        wrow[i] = 0;
        wo[i] = uint32_t((n - c0) * a.pitch) + uint32_t(16 * ((lane & 1) ^ ((r >> 3) & 1)));
      }
    }
    if constexpr (DX) wbase = a.codes + e * a.wrows * a.pitch;
    else wbase = a.codes + (e * a.wrows + c0) * a.pitch;
    const uint32_t wdst = __builtin_amdgcn_readfirstlane(uint32_t(wave) * 1024u);
    // dX scales: 128 bytes a block of 32 columns, BN / 256 blocks of it a wave
    const uint8_t* sbase = nullptr;
    uint32_t so = 0, sdst = 0;
    constexpr int kSLanes = BN / 32;  // of a wave
    if constexpr (DX) {
      sbase = a.scales + e * (a.pitch / 16) * a.np * 2;
      int64_t blk = c0 / 32 + (kSLanes / 8) * wave + ((lane & (kSLanes - 1)) >> 3);
      blk = blk < a.pitch / 16 ? blk : a.pitch / 16 - 1;
      so = uint32_t(blk * a.np * 2) + uint32_t(16 * (lane & 7));
      sdst = __builtin_amdgcn_readfirstlane(uint32_t(16 * kSLanes * wave));
    }
    // step j of this split: its plane and step of the plane
    auto place = [&](int j, int& plane, int& kk) {
      const int t = kbeg + (j < nk ? j : nk - 1);  // past the end: the last step again, never used
      plane = a.planes == 1 ? 0 : t / a.nk;
      kk = t - plane * a.nk;
    };
    auto load_x_part = [&](int j, int i0, int i1) {
      int plane, kk;
      place(j, plane, kk);
      const uint8_t* p = xbase + plane * a.plane + int64_t(kk) * 128;
      const uint32_t dst = uint32_t(j % T::kXRing) * T::kXBytes + xdst;
#pragma unroll
      for (int i = 0; i < T::kXLoads; ++i)
        if (i >= i0 && i < i1) dma16(p, xo[i], dst + 1024u * i);
    };
    auto load_x = [&](int j) { load_x_part(j, 0, T::kXLoads); };
    // the loads of a step go out in parts, between its products
    constexpr int kHalfX = (T::kXLoads + 1) / 2;
    auto load_w = [&](int j) {
      int plane, kk;
      place(j, plane, kk);
      const uint32_t dst = T::kWOff + uint32_t(j % T::kWRing) * T::kWBytes + wdst;
      if constexpr (DX) {
        const uint8_t* p = wbase + int64_t(kk) * kMgStep * a.pitch;
        const int64_t left = a.wrows - 1 - int64_t(kk) * kMgStep;  // rows past the last: the last again, times zero
        const uint32_t most = left < kMgStep ? uint32_t(left) : uint32_t(kMgStep);
#pragma unroll
        for (int i = 0; i < T::kWLoads; ++i)
          dma16(p, (wrow[i] < most ? wrow[i] : most) * uint32_t(a.pitch) + wo[i], dst + 8192u * i);
        const uint32_t sd = T::kSOff + uint32_t(j % T::kWRing) * T::kSBytes + sdst;
        if (lane < kSLanes) dma16(sbase + int64_t(kk) * 128, so, sd);
      } else {
        const uint8_t* p = wbase + int64_t(kk) * 32;
#pragma unroll
        for (int i = 0; i < T::kWLoads; ++i) dma16(p, wo[i], dst + 8192u * i);
      }
    };

    // operand reads
    uint32_t xr[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) xr[s] = swz(uint32_t(32 * MB * wm + i32), uint32_t(4 * q + s));
    u32x4 xf[2][MB];
    auto read_x = [&](u32x4 (&o)[MB], int j, int s) {
      const uint8_t* p = lds + (j % T::kXRing) * T::kXBytes;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
        o[mb] = *reinterpret_cast<const u32x4*>(p + (T::kShare == 1 ? xr[s] : swz(uint32_t(i32), uint32_t(4 * q + s))) + 4096 * mb);
    };
    auto mma = [&](const u32x4 (&w)[NB], const u32x4 (&x)[MB]) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[mb][nb] = mfma32x32x16<XT>(w[nb], x[mb], acc[mb][nb]);
    };

    if constexpr (!DX) {
      uint32_t wr[NB];
      __amdgpu_buffer_rsrc_t srsrc;
      uint32_t soff[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint32_t r = uint32_t(32 * NB * wn + 32 * nb + i32);
        wr[nb] = T::kWOff + 32u * r + 16u * (uint32_t(q) ^ ((r >> 3) & 1u));
        const int64_t n = c0 + r < a.wrows ? c0 + r : a.wrows - 1;
        soff[nb] = uint32_t((n - c0) * (a.pitch / 16));
      }
      {
        const int64_t rows = a.wrows - c0 < BN ? a.wrows - c0 : BN;
        srsrc = buffer_rsrc(a.scales + (e * a.wrows + c0) * (a.pitch / 16), uint32_t(rows * (a.pitch / 16)));
      }
      u32x4 wraw[NB], sc[NB], scn[NB];
      auto read_w = [&](int j) {
        const uint32_t o = uint32_t(j % T::kWRing) * T::kWBytes;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) wraw[nb] = *reinterpret_cast<const u32x4*>(lds + o + wr[nb]);
      };
      // 8 steps' scales from step kk of the plane (past the tile's rows: zeros, never used); the lane's
      // block of an even step is then in the low byte, of an odd one in the third
      auto load_s = [&](u32x4 (&o)[NB], int kk) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[nb] = buf_load16(srsrc, soff[nb] + 2u * uint32_t(kk));
      };
      load_x(0), load_w(0);
      int plane, kk;
      place(0, plane, kk);
      load_s(sc, kk);
      load_s(scn, kk + 8 < a.nk ? kk + 8 : 0);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sc[nb] = u32x4{sc[nb].x >> 8 * q, sc[nb].y >> 8 * q, sc[nb].z >> 8 * q, sc[nb].w >> 8 * q};
#pragma unroll
      for (int p = 1; p < T::kAhead; ++p) {
        load_x(p);
        load_w(p);
      }
      step_barrier<(T::kAhead - 1) * T::kLoads>();
      read_x(xf[0], 0, 0);
      read_w(0);
      int left = (a.nk - kk < 8 ? a.nk - kk : 8);  // steps that sc is good for
      for (int j0 = 0; j0 < nk; j0 += T::kSteps) {  // (a split's steps are even in number)
        // the steps up to the next barrier's first have landed
        step_barrier<(T::kAhead - T::kSteps - 1) * T::kLoads>();
#pragma unroll
        for (int u = 0; u < T::kSteps; ++u) {
          const int j = j0 + u;
          if (left == 0) {
            // the waits on these loads, 8 steps old, come before the step's own loads
            left = a.nk - kk < 8 ? a.nk - kk : 8;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              sc[nb] = u32x4{scn[nb].x >> 8 * q, scn[nb].y >> 8 * q, scn[nb].z >> 8 * q, scn[nb].w >> 8 * q};
              asm volatile("" : "+v"(sc[nb].x), "+v"(sc[nb].y), "+v"(sc[nb].z), "+v"(sc[nb].w));
            }
            load_s(scn, kk + 8 < a.nk ? kk + 8 : 0);
          }
          float scale[NB];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) scale[nb] = mx_scale((sc[nb].x >> (16 * (kk & 1))) & 255u);
          --left;
          if (kk & 1) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) sc[nb] = u32x4{sc[nb].y, sc[nb].z, sc[nb].w, 0u};
          }
          if (++kk == a.nk) kk = 0;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            u32x4 w[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) w[nb] = mx_decode8<XT>(wraw[nb][s], scale[nb]);
            if (s < 3) {
              read_x(xf[(s + 1) & 1], j, s + 1);
            } else {
              read_x(xf[0], j + 1, 0);
              read_w(j + 1);
            }
            // (as it is written, but for 64 rows: 0.65 us a step of 128 x 256 so, 0.73 as the compiler mixes it; of 64
            // rows 0.41 as the compiler mixes it)
            if constexpr (BM > 64) __builtin_amdgcn_sched_barrier(0);
            mma(w, xf[s & 1]);
            if constexpr (BM > 64) __builtin_amdgcn_sched_barrier(0);
            if (s == 0) load_x_part(j + T::kAhead, 0, kHalfX);
            if (s == 1) load_x_part(j + T::kAhead, kHalfX, T::kXLoads);
            if (s == 2) load_w(j + T::kAhead);
          }
        }
      }
    } else {
      // transposing reads: lanes 16 g .. of a group read rows 4 h + j (j = lane / 4 % 4) of the lane half's
      // eight, 8 bytes c = lane % 4 of 32-byte piece 2 wn + g % 2
      uint32_t tr[4][2];
      const int jr = (lane >> 2) & 3, cg = (lane >> 4) & 1;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 32 * q + 8 * s + 4 * h + jr;
          const int f = T::kWRow == 128 ? (r >> 1) & 3 : r & 7;
          tr[s][h] = T::kWOff + uint32_t(r * T::kWRow + 32 * ((2 * wn + cg) ^ f) + 8 * (lane & 3));
        }
      const uint32_t sr = T::kSOff + uint32_t(128 * (4 * wn + (i32 >> 3)) + 64 * q);
      load_w(0);
      load_x(0), load_x(1);
      load_w(1);
      load_x(2);
      step_barrier<T::kLoads>();
      read_x(xf[0], 0, T::kShare == 1 ? 0 : 2 * part);
      for (int j = 0; j < nk; ++j) {
        step_barrier<T::kLoads>();
        const uint32_t wb = uint32_t(j % T::kWRing) * T::kWBytes, sb = uint32_t(j % T::kWRing) * T::kSBytes;
#pragma unroll
        for (int g = 0; g < 4 / T::kShare; ++g) {
          const int s = T::kShare == 1 ? g : 2 * part + g;  // the quarter
          const u32x4 sv = *reinterpret_cast<const u32x4*>(lds + sb + sr + 16 * s);
          u32x4 w[NB];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t at = T::kShare == 1 ? tr[s][h] : tr[g][h] + 2u * 8u * uint32_t(T::kWRow * part);
            const s16x4 t4 =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + wb + at));
            const u32x2 v = __builtin_bit_cast(u32x2, t4);
#pragma unroll
            for (int p = 0; p < 2; ++p) {  // rows 4 h + 2 p, + 1
              const uint32_t two = sv[2 * h + p];
              const float s0 = u2f(two << 16), s1 = u2f(two & 0xFFFF0000u);
              const uint32_t a01 = mx_pair<XT, 0>(v[p], s0), a23 = mx_pair<XT, 1>(v[p], s0);
              const uint32_t b01 = mx_pair<XT, 2>(v[p], s1), b23 = mx_pair<XT, 3>(v[p], s1);
              w[0][2 * h + p] = __builtin_amdgcn_perm(b01, a01, 0x05040100u);
              w[1][2 * h + p] = __builtin_amdgcn_perm(b01, a01, 0x07060302u);
              w[2][2 * h + p] = __builtin_amdgcn_perm(b23, a23, 0x05040100u);
              w[3][2 * h + p] = __builtin_amdgcn_perm(b23, a23, 0x07060302u);
            }
          }
          constexpr int kLast = 4 / T::kShare - 1;
          if (g < kLast) read_x(xf[(g + 1) & 1], j, s + 1);
          else read_x(xf[0], j + 1, T::kShare == 1 ? 0 : 2 * part);
          __builtin_amdgcn_sched_barrier(0);
          mma(w, xf[g & 1]);
          __builtin_amdgcn_sched_barrier(0);
          if (g == 0) load_w(j + 2);
          if (g == (kLast > 0)) load_x_part(j + 3, 0, kHalfX);
          if (g == (kLast > 1 ? 2 : kLast)) load_x_part(j + 3, kHalfX, T::kXLoads);
        }
      }
    }
    wait_vmcnt<0>();  // no load may still be landing in LDS when it holds the output
  }
  __syncthreads();

  if constexpr (T::kShare == 2) {
    // block 1 - part of this wave's sums to its partner, whose own are added: wave `part` ends with block `part`
    const int other = wave ^ (8 / T::kShare);
    f32x4* to = reinterpret_cast<f32x4*>(lds + wave * T::kSwapWave);
    const f32x4* from = reinterpret_cast<const f32x4*>(lds + other * T::kSwapWave);
    f32x16 sum[1][NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[0][nb][r] = part ? acc[1][nb][r] : acc[0][nb][r];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f32x4 v;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = part ? acc[0][nb][4 * r + c] : acc[1][nb][4 * r + c];
        to[64 * (4 * nb + r) + lane] = v;
      }
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 v = from[64 * (4 * nb + r) + lane];
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[0][nb][4 * r + c] = __fadd_rn(sum[0][nb][4 * r + c], v[c]);
      }
    __syncthreads();
    mx_output<XT, DX, 1, NB, OUT32>(a, sum, lds + wave * T::kOutWave, lane, e, live, split, slot0, count, 32 * part,
                                    c0 + 32 * NB * wn);
  } else {
    mx_output<XT, DX, MB, NB, OUT32>(a, acc, lds + wave * T::kOutWave, lane, e, live, split, slot0, count, 32 * MB * wm,
                                     c0 + 32 * NB * wn);
  }
}

// TAIL: no splits; tiles past the last whole round of compute units run as halves of their rows where these take
// one round (a half tile's step takes 0.55 of a whole one's; 896 tiles of 4096 x 4096 x 14336: 3 % less, 2048 tokens' experts 5).  Tiles
// of at most half their rows run as one half (experts 1 to 5 % less; one weight's dX, where it is one tile of each column,
// 0 to 5 % more: not there).
template <int XT, bool DX, int BM, bool OUT32, bool TAIL>
__global__ __launch_bounds__(kMgThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mx4_gemm_kernel(MxGemmArgs a) {
  static_assert(!TAIL || MgTile<DX, BM>::BN == MgTile<DX, BM / 2>::BN, "halves have the tile's columns");
  constexpr int kLds = TAIL && MgTile<DX, BM / 2>::kLds > MgTile<DX, BM>::kLds ? MgTile<DX, BM / 2>::kLds : MgTile<DX, BM>::kLds;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
  lds_escapes(lds);
  int rows = a.row_tiles;  // a plan's: those in use
  if (a.rows.p) rows = a.rows.p[BM == 64 ? 0 : BM == 128 ? 3 : 4];
  const int G = rows * a.col_tiles;
  // An XCD (workgroup % 8) takes a run of tiles, groups of four row tiles walked column by column.
  auto run = [](int t, int n) { return t < n / 8 * 8 ? (t & 7) * (n / 8) + (t >> 3) : t; };
  int t = blockIdx.x, half = -1;
  const int rest = G % a.cus;
  if (TAIL && 2 * rest <= a.cus) {
    if (t >= G + rest) return;
    if (t < G - rest) {
      t = run(t, G - rest);
    } else {
      const int v = run(t - (G - rest), 2 * rest);
      t = G - rest + (v >> 1);
      half = v & 1;
    }
  } else {
    if (t >= G) return;
    t = run(t, G);
  }
  constexpr int GM = 4;
  const int per = GM * a.col_tiles, grp = t / per, r = t - grp * per;
  const int gm = rows - grp * GM < GM ? rows - grp * GM : GM;
  MgRows R = mg_rows<BM>(a, grp * GM + r % gm);
  const int ct = r / gm;
  if constexpr (TAIL) {
    if (half >= 0) {
      R.slot0 += half * (BM / 2);
      R.count -= half * (BM / 2);
      if (R.count <= 0) return;
      if (R.count > BM / 2) R.count = BM / 2;
    }
    if (half >= 0 || (R.count <= BM / 2 && (!DX || a.rows.p))) {
      mg_tile<XT, DX, BM / 2, OUT32>(a, lds, R, ct);
      return;
    }
  }
  mg_tile<XT, DX, BM, OUT32>(a, lds, R, ct);
}

// ---------------------------------------------------------------------------
// Rows as the kernel reads them: 16 bits, 16-byte aligned, zeros up to `pitch` values;
// fp32 rows in three planes of bf16 parts (least first).  by_slot: in the plan's order.
// ---------------------------------------------------------------------------
struct MxRowsArgs {
  const void* x;
  int64_t ld, cols;
  int64_t out_rows, pitch;
  int64_t plane;  // values
  RowsPlan rows;
  int xdiv;
  bool by_slot;
  uint16_t* out;
};

// SPLIT: fp32 rows as three planes, else as they are.  256 threads, workgroup (bx, by) of by_all rows of workgroups.
template <int XT, bool SPLIT>
__device__ __forceinline__ void mx4_rows(const MxRowsArgs& a, unsigned bx, unsigned by, unsigned by_all) {
  typedef typename Elem<XT>::T T;
  constexpr int V = Elem<XT>::kVec, P = 8 / V;
  const int64_t per = a.pitch / 8;
  for (int64_t r = by; r < a.out_rows; r += by_all) {
    int64_t row = r;
    if (a.by_slot) {
      if (a.rows.p && plan_tile(a.rows, int(r / kTileRows)).count <= r % kTileRows) continue;
      row = plan_row(a.rows, r) / a.xdiv;
    }
    const int64_t c8 = int64_t(bx) * 256 + threadIdx.x;
    if (c8 >= per) continue;
    const T* p = static_cast<const T*>(a.x) + row * a.ld + 8 * c8;
    u32x4 v[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int64_t left = a.cols - 8 * c8 - V * j;
      v[j] = left > 0 ? load16_part<XT>(p + V * j, left) : u32x4{0u, 0u, 0u, 0u};
    }
    T* whole = reinterpret_cast<T*>(a.out) + r * a.pitch + 8 * c8;
    if constexpr (XT == RQ_DTYPE_F32 && SPLIT) {
      uint16_t* o = a.out + r * a.pitch + 8 * c8;
      u32x4 h, m, l;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Split3 e = mx_split(u2f(v[j >> 1][2 * (j & 1)])), d = mx_split(u2f(v[j >> 1][2 * (j & 1) + 1]));
        h[j] = e.hi >> 16 | d.hi;
        m[j] = e.mid >> 16 | d.mid;
        l[j] = e.lo >> 16 | d.lo;
      }
      *reinterpret_cast<u32x4*>(o) = l;
      *reinterpret_cast<u32x4*>(o + a.plane) = m;
      *reinterpret_cast<u32x4*>(o + 2 * a.plane) = h;
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) *reinterpret_cast<u32x4*>(whole + V * j) = v[j];
    }
  }
}

template <int XT, bool SPLIT>
__global__ __launch_bounds__(256) void mx4_rows_kernel(MxRowsArgs a) {
  mx4_rows<XT, SPLIT>(a, blockIdx.x, blockIdx.y, gridDim.y);
}

// Scales for dX: bytes [E][N][nb] to bf16 [E][nb][np], 1.0 past N, 64 x 64 a workgroup.
struct MxScalesArgs {
  const uint8_t* in;
  uint16_t* out;
  int64_t N, nb, np;
  unsigned gx, gy, all;  // pieces along n and the blocks, and in all
};
__device__ __forceinline__ void mx4_scales(const MxScalesArgs& a, unsigned first, unsigned step) {
  __shared__ uint8_t t[64][68];
  for (unsigned piece = first; piece < a.all; piece += step) {
    const int64_t n0 = int64_t(piece % a.gx) * 64, b0 = int64_t(piece / a.gx % a.gy) * 64, e = piece / a.gx / a.gy;
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i / 16, c = 4 * (i % 16);  // nb is a multiple of 4
      uint32_t v = 0x7F7F7F7Fu;
      if (n0 + r < a.N && b0 + c < a.nb) v = *reinterpret_cast<const uint32_t*>(a.in + (e * a.N + n0 + r) * a.nb + b0 + c);
      *reinterpret_cast<uint32_t*>(&t[r][c]) = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      const int b = i / 32, r = 2 * (i % 32);
      if (b0 + b >= a.nb || n0 + r >= a.np) continue;  // np is a multiple of 64
      *reinterpret_cast<uint32_t*>(a.out + (e * a.nb + b0 + b) * a.np + n0 + r) = uint32_t(t[r][b]) << 7 | uint32_t(t[r + 1][b]) << 23;
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(256) void mx4_scales_kernel(MxScalesArgs a) { mx4_scales(a, blockIdx.x, gridDim.x); }

// Both, in one launch (4 us of a small call's time): workgroups 0 .. scales - 1, then the rows'.
template <int XT>
__global__ __launch_bounds__(256) void mx4_scales_rows_kernel(MxScalesArgs s, MxRowsArgs r, unsigned scales, unsigned gx, unsigned gy) {
  if (blockIdx.x < scales) {
    mx4_scales(s, blockIdx.x, scales);
  } else {
    const unsigned b = blockIdx.x - scales;
    mx4_rows<XT, true>(r, b % gx, b / gx, gy);
  }
}

// y[t] = RND(sum over its rows, and over the splits of each, in that order)
template <int XT>
__global__ __launch_bounds__(256) void mx4_sum_kernel(MxSumArgs a) {
  const int64_t c = 4 * (int64_t(blockIdx.x) * 256 + threadIdx.x);
  if (c >= a.cols) return;
  for (int64_t t = blockIdx.y; t < a.out_rows; t += gridDim.y) {
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = 0; j < a.ysum; ++j)
      for (int p = 0; p < a.splits; ++p) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + (int64_t(p) * a.M + t * a.ysum + j) * a.ld + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = __fadd_rn(s[i], v[i]);
      }
    typename Elem<XT>::T* p = static_cast<typename Elem<XT>::T*>(a.y) + t * a.ldy + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < a.cols) p[i] = from_f32<XT>(s[i]);
  }
}

// ---- host side -----------------------------------------------------------------
struct MgPlan {
  int bm;
  int splits;
  bool copy, by_slot, partial;  // copy: of the rows
  int planes;
  int64_t xpitch;     // values of a row as the kernel reads it
  int64_t xrows;
  int64_t np, ld;     // dX scales' row, partial sums' row
  int64_t x_bytes, s_bytes, part_bytes;
  int row_tiles, col_tiles;
};

// What a call runs as: a function of its sizes, dtype, row stride and its rows' alignment.
MgPlan mg_plan(const MxCall& c, int cus) {
  MgPlan p{};
  const int64_t wp = mx_pad(c.wk);
  const int64_t cols = c.dx ? c.wk : c.N;
  const int64_t steps64 = c.dx ? ceil_div(c.N, kMgStep) : wp / kMgStep;
  p.planes = c.dt == RQ_DTYPE_F32 ? 3 : 1;
  p.xpitch = steps64 * kMgStep;
  const int64_t xrows = ceil_div(c.M, c.xdiv);
  const bool shared = c.rows.p != nullptr;
  // the rows as they are: 16 bits, whole steps, aligned, within 32-bit offsets of the tile's (a
  // plan's rows: of the first) row; else a copy, in the plan's order where that is too large as well
  const int64_t far = int64_t(1) << 32;
  auto near = [&](int64_t ld) { return (shared ? xrows : 256) * ld * 2 < far; };
  p.copy = p.planes > 1 || c.K != p.xpitch || !c.aligned16 || !near(c.ldx);
  p.by_slot = !shared || (p.copy && !near(p.xpitch));
  p.xrows = shared && p.by_slot ? c.rows.slots() : xrows;
  p.x_bytes = p.copy ? up256(p.planes * p.xrows * p.xpitch * 2) : 0;
  p.np = ceil_div(c.N, kMgStep) * kMgStep;
  p.s_bytes = c.dx ? up256(c.E * (wp / kMxBlock) * p.np * 2) : 0;
  // A copy that is read by slot is as long as its rows: the tile's rows are those that 32-bit offsets reach
  // (64 always are, check_sizes).
  auto reached = [&](int bm) { return !p.copy || !p.by_slot || mx_rows_reached(c.M < bm ? c.M : bm, p.xpitch); };
  // Rows of a tile, and splits of the contraction where the tiles leave compute units idle: the least of an
  // estimate from measured times (us, each within 15 %): a launch, a step, a step's lengthening when all units
  // work; a split's partial sums written and read at 4 TB/s by one more launch.  Forward 128 x 4096 -> 4096: 34,
  // 26, 21 us with 64 rows and 1, 2, 4 splits, 48, 35, 27 with 128, 86, 55, 39 with 256.
  const int64_t groups = shared ? (c.E < c.M ? c.E : c.M) : 1;
  const int64_t steps = p.planes * steps64;
  double best = 0.0;
  p.bm = 64;
  p.splits = 1;
  p.col_tiles = int(ceil_div(cols, c.dx ? 512 : 256));
  for (int bm = 64; bm <= (c.dx ? 128 : 256) && (bm == 64 || reached(bm)); bm *= 2) {
    const double launch = c.dx ? 10.0 : bm == 64 ? 5.0 : bm == 128 ? 7.0 : 8.0;
    // a step of `units` workgroups on the compute units
    auto step = [&](int b, int64_t units) {
      const double alone = c.dx ? (b == 64 ? 0.92 : 1.43) : b == 64 ? 0.41 : b == 128 ? 0.65 : 1.2;
      const double busy = c.dx || b == 256 ? 0.25 : b == 128 ? 0.35 : 0.4;
      return alone * (1.0 + busy * (units < cus ? double(units) / cus : 1.0));
    };
    // experts: about half a tile more each, a whole one for each that has fewer rows than a tile
    const double each = double(c.M) / double(groups);
    const double ends = shared ? double(groups) * (each >= bm ? 0.5 : 1.0 - 0.5 * each / bm) : 0.0;
    const int64_t ct = ceil_div(cols, c.dx ? 512 : 256), tiles = (ceil_div(c.M, bm) + int64_t(ends)) * ct;
    for (int s = 1; s <= 16 && (s == 1 || steps / s >= 4); s *= 2) {
      const int64_t units = tiles * s, rest = units % cus;
      double rounds = double(units / cus) * step(bm, cus);
      if (rest > 0) rounds += s == 1 && bm > 64 && 2 * rest <= cus ? step(bm / 2, 2 * rest) : step(bm, units);
      const double sums = s > 1 || c.ysum > 1 ? 4.0 + double(s) * double(c.M) * double(cols) * 8.0 / 4e6 : 0.0;
      const double t = launch + rounds * double(ceil_div(steps, s)) + sums;
      if (best == 0.0 || t < best) {
        best = t;
        p.bm = bm;
        p.splits = s;
      }
    }
  }
  p.row_tiles = int(!shared ? ceil_div(c.M, p.bm) : p.bm == 64 ? c.rows.T : c.rows.bigs(p.bm == 128 ? 0 : 1));
  p.partial = p.splits > 1 || c.ysum > 1;
  p.ld = (cols + 3) / 4 * 4;
  p.part_bytes = p.partial ? up256(int64_t(p.splits) * c.M * p.ld * 4) : 0;
  return p;
}

template <int XT, bool DX, int BM>
void mg_launch(const MxGemmArgs& a, bool out32, hipStream_t stream) {
  const unsigned tiles = unsigned(a.row_tiles) * unsigned(a.col_tiles);
  const dim3 grid(tiles, unsigned(a.splits));
  if constexpr (BM > 64) {
    if (a.splits == 1) {
      // a tile's halves are two workgroups
      const dim3 all(tiles + unsigned(a.cus));
      if (out32) mx4_gemm_kernel<XT, DX, BM, true, true><<<all, kMgThreads, 0, stream>>>(a);
      else mx4_gemm_kernel<XT, DX, BM, false, true><<<all, kMgThreads, 0, stream>>>(a);
    } else {
      mx4_gemm_kernel<XT, DX, BM, true, false><<<grid, kMgThreads, 0, stream>>>(a);  // partial sums
    }
  } else {
    if (out32) mx4_gemm_kernel<XT, DX, BM, true, false><<<grid, kMgThreads, 0, stream>>>(a);
    else mx4_gemm_kernel<XT, DX, BM, false, false><<<grid, kMgThreads, 0, stream>>>(a);
  }
}

template <int XT>
void mg_launch(const MxGemmArgs& a, bool dx, int bm, bool out32, hipStream_t stream) {
  if (dx) {
    if (bm == 64) mg_launch<XT, true, 64>(a, out32, stream);
    else mg_launch<XT, true, 128>(a, out32, stream);
  } else {
    if (bm == 64) mg_launch<XT, false, 64>(a, out32, stream);
    else if (bm == 128) mg_launch<XT, false, 128>(a, out32, stream);
    else mg_launch<XT, false, 256>(a, out32, stream);
  }
}

dim3 rows_grid(int64_t rows, int64_t pitch) {
  return dim3(unsigned(ceil_div(pitch / 8, 256)), unsigned(rows < 32768 ? rows : 32768));
}

}  // namespace

void mx4_rows_whole(const void* x, int dt, int64_t rows, int64_t cols, int64_t ld, void* out, int64_t pitch, hipStream_t stream) {
  const MxRowsArgs r{x, ld, cols, rows, pitch, 0, RowsPlan{}, 1, false, static_cast<uint16_t*>(out)};
  RQ_DISPATCH_DT(dt, XT, mx4_rows_kernel<XT, false><<<rows_grid(rows, pitch), 256, 0, stream>>>(r));
}

void mx4_sum(const MxSumArgs& s, int dt, hipStream_t stream) {
  const dim3 grid(unsigned(ceil_div(s.ld / 4, 256)), unsigned(s.out_rows < 32768 ? s.out_rows : 32768));
  RQ_DISPATCH_DT(dt, XT, mx4_sum_kernel<XT><<<grid, 256, 0, stream>>>(s));
}

int64_t mx4_gemm_scratch(const MxCall& c, int cus) {
  const MgPlan p = mg_plan(c, cus);
  return p.x_bytes + p.s_bytes + p.part_bytes;
}

void mx4_gemm_tiles(const MxCall& c, int cus, int32_t* out) {
  const MgPlan p = mg_plan(c, cus);
  out[0] = p.bm;
  out[1] = p.splits;
  out[2] = p.copy;
}

int mx4_gemm_run(const MxCall& c, int cus) {
  const MgPlan p = mg_plan(c, cus);
  if (int64_t(p.row_tiles) * p.col_tiles > (int64_t(1) << 22)) return RQ_ERR_UNSUPPORTED;
  uint8_t* ws = static_cast<uint8_t*>(c.scratch);
  const int64_t wp = mx_pad(c.wk);
  MxGemmArgs a{};
  a.x = static_cast<const uint8_t*>(c.x);
  a.ldx = c.ldx * 2;
  a.planes = p.planes;
  a.xdiv = c.xdiv;
  a.by_slot = p.by_slot;
  a.rows = c.rows;
  MxRowsArgs r{};
  const dim3 rgrid = rows_grid(p.xrows, p.xpitch);
  if (p.copy) {
    r = MxRowsArgs{c.x, c.ldx, c.K, p.xrows, p.xpitch, p.xrows * p.xpitch, c.rows, c.xdiv, c.rows.p && p.by_slot,
                   reinterpret_cast<uint16_t*>(ws)};
    a.x = ws;
    a.ldx = p.xpitch * 2;
    a.plane = p.xrows * p.xpitch * 2;
    ws += p.x_bytes;
    if (!c.dx) RQ_DISPATCH_DT(c.dt, XT, mx4_rows_kernel<XT, true><<<rgrid, 256, 0, c.stream>>>(r));
  }
  a.codes = c.codes;
  a.scales = c.scales;
  a.wrows = c.N;
  a.pitch = wp / 2;
  a.np = p.np;
  if (c.dx) {
    const int64_t nb = wp / kMxBlock;
    const MxScalesArgs s{c.scales, reinterpret_cast<uint16_t*>(ws), c.N, nb, p.np, unsigned(p.np / 64), unsigned(ceil_div(nb, 64)),
                         unsigned(p.np / 64 * ceil_div(nb, 64) * c.E)};
    constexpr unsigned kMost = 1u << 22;  // workgroups of either
    const unsigned scales = s.all < kMost ? s.all : kMost, gy = rgrid.y < kMost / rgrid.x ? rgrid.y : kMost / rgrid.x;
    if (!p.copy) mx4_scales_kernel<<<scales, 256, 0, c.stream>>>(s);
    else
      RQ_DISPATCH_DT(c.dt, XT,
                     mx4_scales_rows_kernel<XT><<<scales + rgrid.x * gy, 256, 0, c.stream>>>(s, r, scales, rgrid.x, gy));
    a.scales = ws;
    ws += p.s_bytes;
  }
  a.cols = c.dx ? c.wk : c.N;
  a.nk = int(p.xpitch / kMgStep);
  a.splits = p.splits;
  a.cus = cus;
  a.row_tiles = p.row_tiles;
  a.col_tiles = p.col_tiles;
  a.bias = c.bias;
  a.bias_dt = c.dt;
  const bool out32 = p.partial || c.dt == RQ_DTYPE_F32;
  a.y = p.partial ? ws : c.y;
  a.ldy = p.partial ? p.ld : c.ldy;
  if (c.dt == RQ_DTYPE_F16) mg_launch<RQ_DTYPE_F16>(a, c.dx, p.bm, out32, c.stream);
  else mg_launch<RQ_DTYPE_BF16>(a, c.dx, p.bm, out32, c.stream);
  if (p.partial) {
    mx4_sum(MxSumArgs{reinterpret_cast<const float*>(ws), c.M, p.ld, p.splits, c.ysum, c.M / c.ysum, a.cols, c.y, c.ldy}, c.dt,
            c.stream);
  }
  return rq_check_launch();
}

}  // namespace rq
