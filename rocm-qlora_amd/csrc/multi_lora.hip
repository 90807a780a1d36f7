// The adapters' products over grouped rows (rq_multi_lora.h).
//
// All of them are bound by memory: a row meets r <= 64 ranks, some 4 r operations a
// byte at most, a tenth of what the matrix cores do in the time the byte takes.
// What bounds them beside HBM is the L1: it serves 64 bytes a cycle when four adjacent
// lanes ask for one piece of 64, but a sixteenth lane's row at a time when every lane asks
// for a row of its own, as operand registers hold a matrix.  So rows are loaded straight
// into operand registers where they pass once, and the factors, which serve many rows, go
// through LDS or are read along their rows.  (Rows and factors read as operand registers hold
// them: 296 us for a training step of 4096 rows, K 4096, N 14336, r 64 on four adapters; in
// whole pieces 212; 167 now, of 411 MB that it cannot do without.)
#include "rq_multi_lora.h"

#include "rq_act8.h"
#include "rq_launch.h"
#include "rq_linear_dev.h"

#include <algorithm>

namespace rq {

constexpr int kMlThreads = 256;
constexpr int kMlWaves = kMlThreads / 64;

// The 16-bit halves of fp32 values: hi = RND(v), lo = RND((v - hi) 2^kLoBits) (none for an
// infinity: inf - inf).  fp16's lo part is scaled: |v - hi| is 16 at most (half a step of 65504),
// so that 2^11 of it is the most that fits, and the smallest step of lo is 2^-35 of v instead of
// 2^-24, where hi's own ends.  bf16 has fp32's exponents.
template <int XT>
constexpr int kLoBits = XT == RQ_DTYPE_F16 ? 11 : 0;
template <int XT>
__device__ __forceinline__ void split16(float v, uint32_t& hi, uint32_t& lo) {
  hi = to_x16<XT>(v);
  const float h = from_x16<XT>(hi);
  lo = to_x16<XT>(fabsf(h) == __builtin_inff() ? 0.0f : (v - h) * float(1 << kLoBits<XT>));
}

// acc + the product with lo parts.
template <int XT>
__device__ __forceinline__ f32x4 mma_lo(const u32x4& a, const u32x4& b, f32x4 acc) {
  if constexpr (kLoBits<XT> == 0) {
    return mma<XT>(a, b, acc);
  } else {
    const f32x4 v = mma<XT>(a, b, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] = __builtin_fmaf(v[q], 1.0f / float(1 << kLoBits<XT>), acc[q]);
    return acc;
  }
}

// Workgroup id -> unit of work, 0 .. n - 1 (n or more: none).  Workgroup ids go round the
// eight XCDs; each gets adjacent units, so that what they share stays in its L2.
constexpr int kXcds = 8;
__device__ __forceinline__ unsigned xcd_unit(unsigned id, unsigned n) {
  return id % kXcds * ((n + kXcds - 1) / kXcds) + id / kXcds;
}
inline unsigned xcd_grid(int64_t n) { return unsigned(ceil_div(n, kXcds) * kXcds); }

// ---- shrink ---------------------------------------------------------------------
// A workgroup takes a tile's rows over a split of K.  Tiles of one or two 16-row blocks: the
// four waves divide the split and meet in LDS, 16 rows at a time, summed in the waves' order;
// a wave holds the blocks times JB blocks of 16 ranks, so that a factor's piece is loaded once
// for the tile.  Tiles of more: a wave takes a block, and the factor is shared through LDS
// (four blocks in a wave's registers left it two steps in flight: 44 us for the 27 below).
//
// Rows and factor go through a wave's own piece of LDS.  Rows and A [r][K]: a step's 64
// bytes of each, loaded by four adjacent lanes, the four pieces exchanged by the row so that
// the lanes of a read meet other banks.  B [N][r] (TURNED), whose rows run across the
// contraction: a step's rows are one piece of memory, copied as it lies (with 32 bytes between
// eight-row groups, so that the four lane groups read other banks) and read back a rank's
// values at a time.
//
// Bound by a workgroup's chain of loads (tile, rows, values, the exchange in LDS) and then by
// HBM: dY B of 3342 rows, N 14336, r 64 27 us (96 MB, 3.5 TB/s; a copy reaches 5.2), x A^T of
// 2610 rows, K 11008, r 12 15 us (57 MB, 3.9 TB/s), of 3342 rows, K 4096, r 64 14 us; 224 rows
// on 64 adapters, K 4096, r 32 9 us (19 MB), 8 rows 4.3.  Two pieces in flight instead of one
// in shrink_blocks changed none of it.
constexpr int kShWaves = 4;
constexpr int kShThreads = 64 * kShWaves;

template <int XT, int JB>
struct ShrinkLds {
  static constexpr int kPitch = 16 * JB + 4;
  static constexpr int kRedFloats = kShWaves * 16 * kPitch;
  // elements of one wave's step, with the gaps
  static constexpr int kGap = 32 / int(sizeof(typename Elem<XT>::T));
  static constexpr int kTurn = Elem<XT>::kStep * 16 * JB + 4 * kGap + 2 * Elem<XT>::kVec;  // whole 16 bytes; the last kVec: no one's
  static constexpr int kRows = 32 * 4 * Elem<XT>::kVec;  // of two blocks of rows, a step
  static constexpr int kTurnFloats = kShWaves * (kTurn + kRows) * int(sizeof(typename Elem<XT>::T)) / 4;
};

template <int XT, int NRB, int JB, bool TURNED>
__device__ __forceinline__ void shrink_body(const ShrinkArgs& a, const Tile& tile, const int (&row)[2], int t, int split, int j0,
                                            float* lds) {
  typedef typename Elem<XT>::T T;
  typedef ShrinkLds<XT, JB> L;
  constexpr int V = Elem<XT>::kVec, kStep = Elem<XT>::kStep;
  constexpr int D = NRB == 1 && !TURNED ? 4 : 2;  // steps in flight
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t slot0 = int64_t(kTileRows) * t;
  const T* s0 = static_cast<const T*>(a.s) + tile.adapter * a.s_adapter;
  const T* xr[NRB];
#pragma unroll
  for (int b = 0; b < NRB; ++b) {
    // the row is asked for along with the tile; past the tile's last, row 0: its sums are not read
    xr[b] = static_cast<const T*>(a.x) + int64_t(row[b] < 0 ? 0 : row[b]) * a.ldx + V * (lane & 3);
  }
  const T* sr[JB];
  bool jlive[JB];
#pragma unroll
  for (int b = 0; b < JB; ++b) {
    const int j = j0 + 16 * b + i16;
    jlive[b] = j < a.r;
  }
  // 16 rows of four pieces: piece p of row m lies at 4 m + (p ^ m / 2)
  const int xput = V * (4 * (lane >> 2) + ((lane ^ lane >> 3) & 3)), xget = V * (4 * i16 + ((g ^ i16 >> 1) & 3));
  // TURNED: a step's pieces of V values.  Up to 64 ranks lie end to end in LDS as in memory;
  // of more, this rank block's 64 of each row.  Lanes without a piece repeat the first and
  // put it past the step.
  const int pitch = a.r <= 64 ? a.r : 64;
  T* turn = reinterpret_cast<T*>(lds) + wave * (L::kTurn + L::kRows);
  T* xl = turn + L::kTurn;
  int put[JB];
  if constexpr (TURNED) {
#pragma unroll
    for (int b = 0; b < JB; ++b) {
      const int f = V * (64 * b + lane);
      const bool on = f < kStep * pitch && (a.r <= 64 || j0 + f % 64 < a.r);
      put[b] = on ? f + f / (V * pitch) * L::kGap : L::kTurn - V;
      sr[b] = s0 + (!on ? 0 : a.r <= 64 ? f : (f / 64) * a.r + j0 + f % 64);
    }
  } else {
#pragma unroll
    for (int b = 0; b < JB; ++b) {
      const int j = j0 + 16 * b + (lane >> 2);
      put[b] = V * 64 * b + xput;
      sr[b] = s0 + int64_t(j < a.r ? j : 0) * a.K + V * (lane & 3);
    }
  }
  f32x4 acc[NRB][JB];
#pragma unroll
  for (int b = 0; b < NRB; ++b)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t per = a.k_per_split / kShWaves;
  const int64_t kb = split * a.k_per_split + wave * per;
  const int64_t ke = std::min<int64_t>(kb + per, a.K);
  u32x4 x[D][NRB], s[D][JB];
  auto load = [&](u32x4 (&xv)[NRB], u32x4 (&sv)[JB], int64_t k) {
#pragma unroll
    for (int b = 0; b < NRB; ++b) xv[b] = load16_any(xr[b] + k);
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      sv[j] = load16_any(sr[j] + (TURNED ? k * a.r : k));
    }
  };
  auto products = [&](const u32x4 (&xv)[NRB], const u32x4 (&sv)[JB]) {
#pragma unroll
    for (int j = 0; j < JB; ++j) *reinterpret_cast<u32x4*>(turn + put[j]) = sv[j];
#pragma unroll
    for (int b = 0; b < NRB; ++b) *reinterpret_cast<u32x4*>(xl + V * 64 * b + xput) = xv[b];
    __builtin_amdgcn_wave_barrier();
    u32x4 xo[NRB];
#pragma unroll
    for (int b = 0; b < NRB; ++b) xo[b] = *reinterpret_cast<const u32x4*>(xl + V * 64 * b + xget);
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      u32x4 f;
      if constexpr (TURNED) {
        const T* p = turn + g * (V * pitch + L::kGap) + 16 * j + i16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (XT == RQ_DTYPE_F32) f[e] = f2u(p[e * pitch]);
          else f[e] = uint32_t(p[2 * e * pitch]) | uint32_t(p[(2 * e + 1) * pitch]) << 16;
        }
      } else {
        f = *reinterpret_cast<const u32x4*>(turn + V * 64 * j + xget);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = jlive[j] ? f[e] : 0u;
#pragma unroll
      for (int b = 0; b < NRB; ++b) acc[b][j] = mma<XT>(xo[b], f, acc[b][j]);
      __builtin_amdgcn_sched_barrier(0);  // one rank block's reads at a time in registers
    }
    __builtin_amdgcn_wave_barrier();  // the next step's copy comes after these reads
  };
  int64_t steps = ke > kb ? (ke - kb) / kStep : 0;
  // more than 64 ranks: the factor's last rows are read with their ends in view
  if (TURNED && a.r > 64 && steps > 0 && kb + steps * kStep == a.K) --steps;
  int64_t k = kb, left = steps;
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < steps) load(x[d], s[d], kb + d * kStep);
#pragma unroll 1
  for (; left >= 2 * D; left -= D, k += D * kStep) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      products(x[d], s[d]);
      load(x[d], s[d], k + (D + d) * kStep);
    }
  }
#pragma unroll
  for (int d = 0; d < 2 * D - 1; ++d) {
    if (d >= left) break;
    products(x[d % D], s[d % D]);
    if (d + D < left) load(x[d % D], s[d % D], k + (D + d) * kStep);
  }
  k = kb + steps * kStep;
  if (k < ke) {  // the end of the rows
#pragma unroll
    for (int b = 0; b < NRB; ++b) x[0][b] = load16_part<XT>(xr[b] + k, ke - k - V * (lane & 3));
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      if constexpr (TURNED) s[0][j] = load16_part<XT>(sr[j] + k * a.r, (a.K - k) * a.r - (sr[j] - s0));
      else s[0][j] = load16_part<XT>(sr[j] + k, ke - k - V * (lane & 3));
    }
    products(x[0], s[0]);
  }
  // register q of lane (i, g) is row 4 g + q, rank i
  float* out = a.part + (int64_t(split) * a.rows.slots() + slot0) * a.rp + j0;
  const int ranks = std::min(16 * JB, a.rp - j0);
#pragma unroll
  for (int b = 0; b < NRB; ++b) {
    __syncthreads();  // the turned steps' and the last block's reads are done
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) lds[(wave * 16 + 4 * g + q) * L::kPitch + 16 * j + i16] = acc[b][j][q];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * ranks; i += kShThreads) {
      const int row = i / ranks, j = i - row * ranks;
      float v = lds[row * L::kPitch + j];
#pragma unroll
      for (int w = 1; w < kShWaves; ++w) v = __fadd_rn(v, lds[(w * 16 + row) * L::kPitch + j]);
      out[int64_t(16 * b + row) * a.rp + j] = v;
    }
  }
}

// A wave a 16-row block, 256 bytes of every row (four steps) at a time: the factor's piece of
// them [16 JB ranks][256 bytes] is shared by the waves, B's (TURNED) transposed on its way;
// 16 bytes between rows, so that the lanes of a read meet other banks.  The next piece's loads
// are in flight over this one's products.
constexpr int kShPiece = 256 + 16;  // bytes of a row in LDS

template <int XT, int JB, bool TURNED>
__device__ __forceinline__ void shrink_blocks(const ShrinkArgs& a, const Tile& tile, int t, int split, int j0, char* lds) {
  typedef typename Elem<XT>::T T;
  constexpr int V = Elem<XT>::kVec, kStep = Elem<XT>::kStep, kPiece = 4 * kStep, P = kShPiece / int(sizeof(T));
  const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t slot0 = int64_t(kTileRows) * t;
  const T* s0 = static_cast<const T*>(a.s) + tile.adapter * a.s_adapter;
  T* sl = reinterpret_cast<T*>(lds);
  T* xl = sl + 16 * JB * P + wave * 16 * P;
  // this lane's loads of the wave's rows: row 4 b + lane / 16, 16 bytes at lane % 16
  const T* xr[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int row = plan_row(a.rows, slot0 + 16 * wave + 4 * b + g);
    xr[b] = static_cast<const T*>(a.x) + int64_t(row < 0 ? 0 : row) * a.ldx + V * i16;
  }
  // of the factor.  A: rank 16 b + tid / 16, 16 bytes at tid % 16.  B: a block of V k and V
  // ranks, one a thread where there are that many: ranks V (tid % n), k V (tid / n), n = 16 JB / V.
  constexpr int kRankBlocks = 16 * JB / V, kBlocks = kRankBlocks * (kPiece / V);
  constexpr int kPer = TURNED ? V : JB;
  const int tr = V * (tid % kRankBlocks), tk = V * (tid / kRankBlocks);
  static_assert(!TURNED || kBlocks <= kShThreads, "a block a thread");
  const bool turns = tid < kBlocks && j0 + tr < a.r;
  auto at = [](int row, int piece) { return V * (piece ^ ((row >> 3) & 7)); };  // of a factor's row
  u32x4 x[4], s[kPer];
  auto load = [&](int64_t k, int64_t end) {  // k .. end - 1 of the piece at k
    // whole pieces; 16 bytes from the last of B's ranks on stay in B
    if (k + kPiece <= end && (!TURNED || a.r % V == 0 || (k + kPiece) * a.r + V <= a.K * a.r)) {
#pragma unroll
      for (int b = 0; b < 4; ++b) x[b] = load16_any(xr[b] + k);
#pragma unroll
      for (int b = 0; b < kPer; ++b) {
        if constexpr (TURNED) {
          s[b] = load16_any(s0 + (turns ? (k + tk + b) * a.r + j0 + tr : 0));
        } else {
          const int j = j0 + 16 * b + (tid >> 4);
          s[b] = load16_any(s0 + int64_t(j < a.r ? j : 0) * a.K + k + V * (tid & 15));
        }
      }
    } else {  // the end of the rows, or of B
#pragma unroll
      for (int b = 0; b < 4; ++b) x[b] = load16_part<XT>(xr[b] + k, end - k - V * i16);
#pragma unroll
      for (int b = 0; b < kPer; ++b) {
        if constexpr (TURNED) {
          s[b] = load16_part<XT>(s0 + (k + tk + b) * a.r + j0 + tr, turns && k + tk + b < end ? a.r - j0 - tr : 0);
        } else {
          const int j = j0 + 16 * b + (tid >> 4);
          s[b] = load16_part<XT>(s0 + int64_t(j < a.r ? j : 0) * a.K + k + V * (tid & 15), end - k - V * (tid & 15));
        }
      }
    }
  };
  auto stage = [&]() {
#pragma unroll
    for (int b = 0; b < 4; ++b) *reinterpret_cast<u32x4*>(xl + (4 * b + g) * P + V * i16) = x[b];
    if constexpr (TURNED) {
      if (tid < kBlocks) {
#pragma unroll
        for (int c = 0; c < V; ++c) {
          u32x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (XT == RQ_DTYPE_F32) o[e] = s[e][c];
            else o[e] = __builtin_amdgcn_perm(s[2 * e + 1][c >> 1], s[2 * e][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
            o[e] = j0 + tr + c < a.r ? o[e] : 0u;
          }
          *reinterpret_cast<u32x4*>(sl + (tr + c) * P + at(tr + c, tk / V)) = o;
        }
      }
    } else {
#pragma unroll
      for (int b = 0; b < JB; ++b) {
        const bool on = j0 + 16 * b + (tid >> 4) < a.r;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[b][e] = on ? s[b][e] : 0u;
        *reinterpret_cast<u32x4*>(sl + (16 * b + (tid >> 4)) * P + at(16 * b + (tid >> 4), tid & 15)) = s[b];
      }
    }
  };
  f32x4 acc[JB];
#pragma unroll
  for (int j = 0; j < JB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t kb = split * a.k_per_split, ke = std::min<int64_t>(kb + a.k_per_split, a.K);
  if (kb < ke) load(kb, ke);
#pragma unroll 1
  for (int64_t k = kb; k < ke; k += kPiece) {
    if (k > kb) __syncthreads();  // the last piece is read
    stage();
    __syncthreads();
    if (k + kPiece < ke) load(k + kPiece, ke);
    if (16 * wave >= tile.count) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u32x4 xo = *reinterpret_cast<const u32x4*>(xl + i16 * P + q * kStep + V * g);
#pragma unroll
      for (int j = 0; j < JB; ++j)
        acc[j] = mma<XT>(xo, *reinterpret_cast<const u32x4*>(sl + (16 * j + i16) * P + at(16 * j + i16, 4 * q + g)), acc[j]);
    }
  }
  if (16 * wave >= tile.count) return;
  // register q of lane (i, g) is row 4 g + q, rank i
  float* out = a.part + (int64_t(split) * a.rows.slots() + slot0 + 16 * wave + 4 * g) * a.rp + j0 + i16;
#pragma unroll
  for (int j = 0; j < JB; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (j0 + 16 * j < a.rp) out[int64_t(q) * a.rp + 16 * j] = acc[j][q];
}

template <int XT, int JB, bool TURNED>
__global__ __launch_bounds__(kShThreads) __attribute__((amdgpu_waves_per_eu(3))) void shrink_kernel(ShrinkArgs a) {
  typedef ShrinkLds<XT, JB> L;
  constexpr int kBlockFloats = (16 * JB + 64) * kShPiece / 4;
  constexpr int kWaveFloats = L::kTurnFloats > L::kRedFloats ? L::kTurnFloats : L::kRedFloats;
  __shared__ __attribute__((aligned(16))) float lds[kWaveFloats > kBlockFloats ? kWaveFloats : kBlockFloats];
  // an XCD's workgroups take one split's piece of the factors, or two
  const unsigned unit = xcd_unit(blockIdx.x, unsigned(a.rows.T) * unsigned(a.splits));
  const int t = int(unit % unsigned(a.rows.T)), split = int(unit / unsigned(a.rows.T));
  if (split >= a.splits) return;
  const int j0 = 16 * JB * int(blockIdx.y);
  const Tile tile = plan_tile(a.rows, t);
  int row[2];  // of the lane's loads: lane / 4 in each 16-row block
#pragma unroll
  for (int b = 0; b < 2; ++b) row[b] = plan_row(a.rows, int64_t(kTileRows) * t + 16 * b + ((threadIdx.x & 63) >> 2));
  if (tile.count == 0 || tile.adapter < 0) return;
  if (tile.count <= 16) shrink_body<XT, 1, JB, TURNED>(a, tile, row, t, split, j0, lds);
  else if (tile.count <= 32) shrink_body<XT, 2, JB, TURNED>(a, tile, row, t, split, j0, lds);
  else shrink_blocks<XT, JB, TURNED>(a, tile, t, split, j0, reinterpret_cast<char*>(lds));
}

// About two workgroups a compute unit, each with four steps a wave (many tiles: eight, since
// every later workgroup of a tile sums the splits; a training step of 4096 rows, K 4096,
// N 14336, r 64, replayed from a graph: 162 - 166 us, with sixteen 168, with twenty-eight 187).
void plan_shrink(int64_t T, int64_t K, int step, int cus, int* splits, int64_t* per) {
  const int64_t unit = int64_t(step) * kShWaves;
  int64_t s = ceil_div(2 * cus, std::max<int64_t>(T, 1));
  s = std::min(s, std::max<int64_t>(K / ((T >= 48 ? 8 : 4) * unit), 1));
  s = std::min<int64_t>(std::max<int64_t>(s, 1), 16);
  *per = ceil_div(ceil_div(K, s), unit) * unit;
  *splits = int(ceil_div(K, *per));
}

template <int XT, bool TURNED>
int run_shrink(const ShrinkArgs& a, hipStream_t stream) {
  const int jb = a.rp <= 16 ? 1 : (a.rp <= 32 ? 2 : 4);
  if (int64_t(a.rows.T) * a.splits > kMaxThreads1D / kShThreads - kXcds) return RQ_ERR_UNSUPPORTED;
  const dim3 grid(xcd_grid(int64_t(a.rows.T) * a.splits), unsigned(ceil_div(a.rp, 16 * jb)));
  if (jb == 1) shrink_kernel<XT, 1, TURNED><<<grid, kShThreads, 0, stream>>>(a);
  else if (jb == 2) shrink_kernel<XT, 2, TURNED><<<grid, kShThreads, 0, stream>>>(a);
  else shrink_kernel<XT, 4, TURNED><<<grid, kShThreads, 0, stream>>>(a);
  return rq_check_launch();
}

// ---- the row sums' operands (their layout: opt_at, rq_multi_lora.h) -----------------
// A tile's operands from LDS, rows of `pitch` (16-bit: hi | lo); zeros past its `count` rows.
template <int XT>
__device__ __forceinline__ void store_operands(typename Elem<XT>::T* opt, const typename Elem<XT>::T* op, int pitch, int rp,
                                               int64_t slot0, int count) {
  typedef typename Elem<XT>::T T;
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4, blocks = rp >> 4;
  for (int k = threadIdx.x >> 6; k < (count > 32 ? 2 : 1) * blocks; k += kMlWaves) {
    const int first = 32 * (k / blocks) + 8 * g, j = 16 * (k % blocks) + i16;
    T* o = opt + opt_at<XT>(slot0 + first, j, rp);
    const T* p = op + first * pitch + j;
    if constexpr (XT == RQ_DTYPE_F32) {
      f32x4 v[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e >> 2][e & 3] = first + e < count ? p[e * pitch] : 0.0f;
      *reinterpret_cast<f32x4*>(o) = v[0];
      *reinterpret_cast<f32x4*>(o + 256) = v[1];
    } else {
      u32x4 hi = u32x4{0u, 0u, 0u, 0u}, lo = hi;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (first + e >= count) break;
        hi[e >> 1] |= uint32_t(p[e * pitch]) << (16 * (e & 1));
        lo[e >> 1] |= uint32_t(p[e * pitch + rp]) << (16 * (e & 1));
      }
      *reinterpret_cast<u32x4*>(o) = hi;
      *reinterpret_cast<u32x4*>(o + 512) = lo;
    }
  }
}

// The splits' sum of a tile's slots, in order, as operands in LDS rows of `pitch`.  A thread
// takes four adjacent ranks of two slots at a time, four splits of each in flight.  Ranks from
// r on are zeros whatever the row held: an infinity times their zero factors is no zero.
template <int XT>
__device__ __forceinline__ void sum_operands(typename Elem<XT>::T* op, int pitch, const float* part, int splits, int64_t slots,
                                             int r, int rp, int64_t slot0, int count) {
  const int quads = rp / 4, items = ((count + 15) & ~15) * quads;
  const int64_t stride = slots * rp;
  const float* p0 = part + slot0 * rp;
  for (int i0 = threadIdx.x; i0 < items; i0 += 2 * kMlThreads) {
    f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    const float* p[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) p[h] = p0 + 4 * (i0 + h * kMlThreads < items ? i0 + h * kMlThreads : i0);  // rows are end to end
    for (int k = 0; k < splits; k += 4) {
      f32x4 q[2][4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (n == 0 || k + n < splits) q[h][n] = *reinterpret_cast<const f32x4*>(p[h] + (k + n) * stride);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (n == 0 || k + n < splits)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[h][e] = __fadd_rn(v[h][e], q[h][n][e]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = i0 + h * kMlThreads;
      if (i >= items) break;
      const int m = i / quads, j = 4 * (i - m * quads);
      typename Elem<XT>::T* o = op + m * pitch + j;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[h][e] = j + e < r ? v[h][e] : 0.0f;
      if constexpr (XT == RQ_DTYPE_F32) {
        *reinterpret_cast<f32x4*>(o) = v[h];
      } else {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split16<XT>(v[h][e], hi[e], lo[e]);
        *reinterpret_cast<u32x2*>(o) = u32x2{hi[0] | hi[1] << 16, hi[2] | hi[3] << 16};
        *reinterpret_cast<u32x2*>(o + rp) = u32x2{lo[0] | lo[1] << 16, lo[2] | lo[3] << 16};
      }
    }
  }
}

// The operands alone, for gradients without one of the rows: a workgroup a tile.
template <int XT>
__global__ __launch_bounds__(kMlThreads) void operands_kernel(OperandsArgs a) {
  typedef typename Elem<XT>::T T;
  extern __shared__ uint32_t operands_lds[];
  T* op = reinterpret_cast<T*>(operands_lds);
  const Tile tile = plan_tile(a.rows, int(blockIdx.x));
  if (tile.count == 0 || tile.adapter < 0) return;
  const int pitch = (XT == RQ_DTYPE_F32 ? a.rp : 2 * a.rp) + Elem<XT>::kVec;
  const int64_t slot0 = int64_t(kTileRows) * blockIdx.x;
  sum_operands<XT>(op, pitch, a.part, a.splits, a.rows.slots(), a.r, a.rp, slot0, tile.count);
  __syncthreads();
  store_operands<XT>(static_cast<T*>(a.opt), op, pitch, a.rp, slot0, tile.count);
}

// Dynamic LDS of a launch: past 64 KiB (ranks above 200) the kernel has to be told.
template <typename K>
int allow_lds(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
  constexpr int kMost = 160 << 10;
  if (bytes <= (64u << 10)) return RQ_OK;
  return bytes > size_t(kMost) ? RQ_ERR_UNSUPPORTED : allow_dynamic_lds(reinterpret_cast<const void*>(kernel), kMost, done);
}

template <int XT>
int run_operands(const OperandsArgs& a, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const int pitch = (XT == RQ_DTYPE_F32 ? a.rp : 2 * a.rp) + Elem<XT>::kVec;
  const size_t bytes = size_t(kTileRows) * pitch * sizeof(typename Elem<XT>::T);
  const int st = allow_lds(operands_kernel<XT>, bytes, done);
  if (st != RQ_OK) return st;
  operands_kernel<XT><<<unsigned(a.rows.T), kMlThreads, bytes, stream>>>(a);
  return rq_check_launch();
}

// ---- expand ---------------------------------------------------------------------
// A workgroup takes a tile: it sums the splits of its slots and keeps them in LDS as operands.
// Its four waves divide the tile's 16-row blocks (1, 2 or 4) and, where there are fewer than
// four, adjacent columns; a wave's step is 16 kVec columns.  The slots are the A operand and
// column kVec i + c of the factor is row i of the B operand of product c, so that a lane ends
// with kVec adjacent columns of rows 4 g + q: 256 bytes of a row by 16 adjacent lanes.
//
// B's rows [N][r] go through LDS, one rank step (32 ranks of 16 bits, 16 of fp32) of all the
// waves' columns at a time, copied as they lie (up to a step of ranks; of more, a step's ranks
// of each row) with 16 bytes between groups of kVec rows, so that the lanes of a read meet
// other banks.  A's rows [r][K] are read along the row and transposed in registers.
//
// Bound by HBM with a base: 4096 rows, N 14336, r 64 56 us (base and result 235 MB, 4.2 TB/s),
// 3001 rows, N 4096, r 12 16 us (3.1 TB/s).  Without one (dX of 4096 rows, K 4096: 22 us,
// 34 MB written) by a workgroup's chain: rows, splits, factor pieces, each waiting for the
// last; there are two workgroups a compute unit, and more of them sum the splits more often.
// Four slots' splits in flight instead of two: no faster.
template <int XT>
struct ExpandLds {
  static constexpr int kCols = 16 * Elem<XT>::kVec;   // of a wave
  // elements of one wave's columns of a rank step, with the gaps
  static constexpr int kStage = kCols * Elem<XT>::kStep + 16 * Elem<XT>::kVec;
};

// kVec columns from `col` on of A's rows j .. j + kVec - 1, and their transpose (zeros for
// ranks from r on).
template <int XT, bool EDGE>
__device__ __forceinline__ void load_ranks(u32x4 (&row)[Elem<XT>::kVec], const typename Elem<XT>::T* s, int64_t C, int64_t col,
                                           int r, int j) {
#pragma unroll
  for (int e = 0; e < Elem<XT>::kVec; ++e) {
    const typename Elem<XT>::T* p = s + int64_t(j + e < r ? j + e : 0) * C + col;
    row[e] = EDGE ? load16_part<XT>(p, C - col) : load16_any(p);
  }
}
template <int XT>
__device__ __forceinline__ void turn_ranks(u32x4 (&f)[Elem<XT>::kVec], const u32x4 (&row)[Elem<XT>::kVec], int r, int j) {
  constexpr int V = Elem<XT>::kVec;
#pragma unroll
  for (int c = 0; c < V; ++c) {
    if constexpr (XT == RQ_DTYPE_F32) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[c][e] = row[e][c];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[c][e] = __builtin_amdgcn_perm(row[2 * e + 1][c >> 1], row[2 * e][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
    }
  }
  if (j + V > r) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t keep;
      if constexpr (XT == RQ_DTYPE_F32) keep = j + e < r ? ~0u : 0u;
      else keep = j + 2 * e + 1 < r ? ~0u : (j + 2 * e < r ? 0xFFFFu : 0u);
#pragma unroll
      for (int c = 0; c < V; ++c) f[c][e] &= keep;
    }
  }
}

// BLOCKS: 16-row blocks that the waves divide (1, 2, 4).  EDGES: there are columns that a
// whole wave does not fill, or ranks of B's rows that 16 bytes run past.  LINES: the results'
// rows are whole 64-byte lines.  BASED: there is a base.
template <int XT, bool FACTOR_ROWS, bool EDGES, bool LINES, bool BASED, int BLOCKS>
__device__ __forceinline__ void expand_body(const ExpandArgs& a, const Tile& tile, int t, int chunk, typename Elem<XT>::T* lds) {
  typedef typename Elem<XT>::T T;
  typedef ExpandLds<XT> L;
  constexpr int V = Elem<XT>::kVec, kStep = Elem<XT>::kStep;
  constexpr int GROUPS = kMlWaves / BLOCKS;                      // of columns
  constexpr int PIECES = FACTOR_ROWS ? GROUPS * L::kCols * kStep / V / kMlThreads : V;
  const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int block = wave % BLOCKS, group = wave / BLOCKS;
  const int64_t slot0 = int64_t(kTileRows) * t;
  const bool adapted = tile.adapter >= 0;
  const int pitch = (XT == RQ_DTYPE_F32 ? a.rp : 2 * a.rp) + V;  // of the slots' operands
  T* op = lds + (FACTOR_ROWS ? GROUPS * L::kStage : 0);
  // 16 ranks of 16 bits: lane groups 2 and 3 take the lo parts, of the same ranks as 0 and 1 (one
  // matrix instruction where lo is not scaled)
  const bool half = XT != RQ_DTYPE_F32 && a.rp < kStep;
  const T* s = static_cast<const T*>(a.s) + (adapted ? tile.adapter : 0) * a.s_adapter;
  const float scale = adapted ? a.scaling[tile.adapter] : 0.0f;
  const int64_t c_first = int64_t(chunk) * a.iters * (kMlWaves * L::kCols);
  const int steps = adapted ? int(ceil_div(a.rp, kStep)) : 1;    // of ranks
  const int sp = a.r < kStep ? a.r : kStep;                      // ranks of a column in LDS
  const float per_sp = 1.0f / float(sp);

  // this lane's rows (past the tile's last: -1)
  int row[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) row[q] = plan_row(a.rows, slot0 + 16 * block + 4 * g + q);
  // a step's pieces of B, as this thread copies them (32-bit offsets from a uniform address),
  // or of A, as its lane uses them
  u32x4 piece[PIECES];
  uint32_t off[FACTOR_ROWS ? PIECES : 1], put[FACTOR_ROWS ? PIECES : 1];
  if constexpr (FACTOR_ROWS) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int f = V * (tid + kMlThreads * k);
      off[k] = uint32_t(a.r <= kStep ? f : f / kStep * a.r + f % kStep);
      // f / (V sp), exact: the quotient is 1 / (2 sp) or more from an integer
      put[k] = uint32_t(f + int((float(f / V) + 0.5f) * per_sp) * V);
    }
  }
  auto fetch = [&](int64_t c0, int j0) {
    if constexpr (!FACTOR_ROWS) {
      const int64_t col = c0 + group * L::kCols + V * i16;
      load_ranks<XT, EDGES>(piece, s, a.C, col < a.C ? col : 0, a.r, j0 + (half ? V * (g & 1) : V * g));
    } else {
      const T* from = s + c0 * a.r + j0;
      const int64_t left = (a.C - c0) * a.r - j0;
      const uint32_t end = uint32_t(left < INT32_MAX ? left : INT32_MAX);
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const int f = V * (tid + kMlThreads * k);
        const bool there = a.r <= kStep ? f < GROUPS * L::kCols * sp : j0 + f % kStep < a.r;
        if constexpr (EDGES) piece[k] = load16_part<XT>(from + off[k], there && off[k] < end ? int64_t(end - off[k]) : 0);
        else piece[k] = load16_any(from + (there && off[k] < end ? off[k] : 0u));
      }
    }
  };
  auto stage = [&]() {
    if constexpr (FACTOR_ROWS) {
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const int f = V * (tid + kMlThreads * k);
        if (f < GROUPS * L::kCols * sp) *reinterpret_cast<u32x4*>(lds + put[k]) = piece[k];
      }
    }
  };
  if (adapted) fetch(c_first, 0);
  u32x4 base[4];
  auto fetch_base = [&](int64_t at) {  // from column `at` on
    if constexpr (BASED) {
      if (!EDGES && at - V * i16 >= a.C) at = V * i16;  // not used
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const T* p = static_cast<const T*>(a.base) + (row[q] < 0 ? 0 : row[q]) * a.ld_base + at;
        base[q] = EDGES ? load16_part<XT>(p, a.C - at) : load16_any(p);
      }
    }
  };
  fetch_base(c_first + group * L::kCols + V * i16);
  if (adapted) sum_operands<XT>(op, pitch, a.part, a.splits, a.rows.slots(), a.r, a.rp, slot0, tile.count);
  __syncthreads();
  if (a.opt && adapted && chunk == 0) store_operands<XT>(static_cast<T*>(a.opt), op, pitch, a.rp, slot0, tile.count);
  const bool rows_here = 16 * block < tile.count;
#pragma unroll 1
  for (int it = 0; it < a.iters * BLOCKS; ++it) {
    const int64_t w0 = c_first + int64_t(it) * (GROUPS * L::kCols);  // of the workgroup
    if (w0 >= a.C) return;
    const int64_t c0 = w0 + group * L::kCols, col = c0 + V * i16;
    const bool here = rows_here && c0 < a.C;
    // the next step's pieces (after the last step: these again, so that no branch makes the
    // loads' results wait)
    const int64_t w1 = it + 1 < a.iters * BLOCKS && w0 + GROUPS * L::kCols < a.C ? w0 + GROUPS * L::kCols : w0;
    auto ahead = [&](int k) { fetch(k + 1 < steps ? w0 : w1, k + 1 < steps ? (k + 1) * kStep : 0); };
    f32x4 acc[V];
#pragma unroll
    for (int c = 0; c < V; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (adapted) {
#pragma unroll 1
      for (int k = 0; k < steps; ++k) {
        u32x4 f[V];
        const int j = k * kStep + (half ? V * (g & 1) : V * g);
        if constexpr (FACTOR_ROWS) {
          stage();
          __syncthreads();
          if (BLOCKS > 1) ahead(k);
          const T* p = lds + (group * L::kCols + V * i16) * sp + (group * 16 + i16) * V + (j - k * kStep);
#pragma unroll
          for (int c = 0; c < V; ++c) f[c] = load16_any(p + c * sp);
          if (j + V > a.r) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t keep;
              if constexpr (XT == RQ_DTYPE_F32) keep = j + e < a.r ? ~0u : 0u;
              else keep = j + 2 * e + 1 < a.r ? ~0u : (j + 2 * e < a.r ? 0xFFFFu : 0u);
#pragma unroll
              for (int c = 0; c < V; ++c) f[c][e] &= keep;
            }
          }
        } else {
          turn_ranks<XT>(f, piece, a.r, j);
          ahead(k);
        }
        if (here) {
          const T* u = op + (16 * block + i16) * pitch + k * kStep + V * g;
          u32x4 hi = *reinterpret_cast<const u32x4*>(u);
          u32x4 lo = hi;  // `half`: of lane groups 2 and 3
          const bool apart = XT != RQ_DTYPE_F32 && (!half || kLoBits<XT> > 0);
          if (XT != RQ_DTYPE_F32 && !half) {
            lo = *reinterpret_cast<const u32x4*>(u + a.rp);
          } else if (apart) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              lo[e] = g < 2 ? 0u : lo[e];
              hi[e] = g < 2 ? hi[e] : 0u;
            }
          }
#pragma unroll
          for (int c = 0; c < V; ++c) acc[c] = mma<XT>(hi, f[c], acc[c]);
          if (apart) {
#pragma unroll
            for (int c = 0; c < V; ++c) acc[c] = mma_lo<XT>(lo, f[c], acc[c]);
          }
        }
        if constexpr (FACTOR_ROWS) {
          __syncthreads();
          if (BLOCKS == 1) ahead(k);  // eight pieces: not over the products, for the registers
        }
      }
    }
    float v[4][V];
#pragma unroll
    for (int q = 0; q < 4; ++q) unpack16<XT>(BASED ? base[q] : u32x4{0u, 0u, 0u, 0u}, v[q]);
    fetch_base(w1 + group * L::kCols + V * i16);
    if (!here) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (adapted) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[q][e] = __fadd_rn(v[q][e], __fmul_rn(scale, acc[e][q]));
      }
      if (row[q] < 0) continue;
      T* o = static_cast<T*>(a.out) + row[q] * a.ld_out + col;
      if constexpr (EDGES) store16_part<XT>(o, v[q], a.C - col);
      else store16<LINES>(o, pack16<XT>(v[q]));
    }
  }
}

template <int XT, bool FACTOR_ROWS, bool EDGES, bool LINES, bool BASED>
__global__ __launch_bounds__(kMlThreads) __attribute__((amdgpu_waves_per_eu(EDGES ? 2 : 3))) void expand_kernel(ExpandArgs a) {
  typedef typename Elem<XT>::T T;
  extern __shared__ uint32_t expand_lds[];
  T* lds = reinterpret_cast<T*>(expand_lds);
  const int chunk = int(blockIdx.x % unsigned(a.chunks)), t = int(blockIdx.x / unsigned(a.chunks));
  const Tile tile = plan_tile(a.rows, t);
  if (tile.count == 0) return;
  if (tile.adapter < 0 && a.base == a.out && a.ld_base == a.ld_out) return;  // in place, nothing to add
  if (tile.count <= 16) expand_body<XT, FACTOR_ROWS, EDGES, LINES, BASED, 1>(a, tile, t, chunk, lds);
  else if (tile.count <= 32) expand_body<XT, FACTOR_ROWS, EDGES, LINES, BASED, 2>(a, tile, t, chunk, lds);
  else expand_body<XT, FACTOR_ROWS, EDGES, LINES, BASED, 4>(a, tile, t, chunk, lds);
}

template <int XT, bool FACTOR_ROWS>
int run_expand(ExpandArgs a, int cus, hipStream_t stream) {
  typedef ExpandLds<XT> L;
  constexpr int V = Elem<XT>::kVec, es = int(sizeof(typename Elem<XT>::T));
  const int64_t steps = ceil_div(a.C, int64_t(kMlWaves) * L::kCols);
  // steps of a workgroup: as many as leave eight workgroups a compute unit (both products of
  // 4096 rows, N 14336: 63 - 68 us with four or eight, 71 with two)
  a.iters = int(std::max<int64_t>(1, std::min<int64_t>(8, a.rows.T * steps / (8 * cus))));
  a.chunks = int(ceil_div(steps, a.iters));
  if (int64_t(a.rows.T) * a.chunks > kMaxThreads1D / kMlThreads) return RQ_ERR_UNSUPPORTED;
  // LDS: the staged columns and the operands of 1, 2 or 4 row blocks, whichever is largest
  const int pitch = (es == 4 ? a.rp : 2 * a.rp) + V;
  size_t bytes = 0;
  for (int blocks = 1; blocks <= kMlWaves; blocks *= 2)
    bytes = std::max(bytes, size_t((FACTOR_ROWS ? kMlWaves / blocks * L::kStage : 0) + 16 * blocks * pitch) * es);
  const bool edges = a.C % L::kCols != 0 || (FACTOR_ROWS && a.r > Elem<XT>::kStep && a.r % V != 0);
  const unsigned grid = unsigned(int64_t(a.rows.T) * a.chunks);
  const bool lines = !edges && aligned(a.out, 64) && a.ld_out * es % 64 == 0;
  auto launch = [&](auto kernel, std::atomic<uint64_t>& done) {
    const int st = allow_lds(kernel, bytes, done);
    if (st != RQ_OK) return st;
    kernel<<<grid, kMlThreads, bytes, stream>>>(a);
    return rq_check_launch();
  };
  static std::atomic<uint64_t> done[6];
  if (!a.base) {
    if (edges) return launch(expand_kernel<XT, FACTOR_ROWS, true, false, false>, done[0]);
    return lines ? launch(expand_kernel<XT, FACTOR_ROWS, false, true, false>, done[1])
                 : launch(expand_kernel<XT, FACTOR_ROWS, false, false, false>, done[2]);
  }
  if (edges) return launch(expand_kernel<XT, FACTOR_ROWS, true, false, true>, done[3]);
  return lines ? launch(expand_kernel<XT, FACTOR_ROWS, false, true, true>, done[4])
               : launch(expand_kernel<XT, FACTOR_ROWS, false, false, true>, done[5]);
}

// ---- sums over the rows of an adapter ----------------------------------------------
// D[c][j] = sum_m x[row m][c] u[m][j], the contraction over the slow index of x: lane
// (i, g) loads CW columns of the eight rows of slots 8 g .. 8 g + 7, which byte permutes
// turn into CW operand rows of eight consecutive slots (16-bit; fp32 values are operands
// as they are).  A workgroup takes 16 CW columns over the rows of a chunk, 32 slots a
// step; its four waves take steps in turn and meet in LDS, summed as (0 + 2) + (1 + 3).
// Where a wave holds 64 ranks CW is 4: with 8 the accumulators leave two waves a SIMD (a
// backward pass of 4096 rows, r 64: 97 -> 109 us), and two steps in flight do not fit the
// registers.  dA and dB of 3342 rows, K 4096, N 14336, r 64: 41 us (123 MB of rows, 3.0 TB/s),
// bound by what passes through the L1 (its return path is busy 84 % of the time, its address
// unit 67): at 64 columns by 64 ranks a wave's operands are twice its rows' bytes.  From an
// 8-bit checkpoint of 2048 rows, K = N = 4096, r 16: 11 us.
template <int XT, int CW>
struct ColPiece {
  static constexpr int kWords = XT == RQ_DTYPE_F32 ? CW : CW / 2;
  uint32_t d[kWords];
};

// columns of a lane, by 16-rank blocks of a wave
template <int XT>
constexpr int rowsum_cw(int jb) {
  return XT == RQ_DTYPE_F32 || jb > 2 ? 4 : 8;
}

// CODES: the rows are 8-bit codes with exponents.
template <int XT, int CW, bool CODES>
struct RawPiece {
  uint32_t d[CODES ? CW / 4 : ColPiece<XT, CW>::kWords];
  uint32_t e;  // of codes
};

// full: all CW columns of this lane exist (of codes they do: rows end in whole blocks).
template <int XT, int CW, bool CODES>
__device__ __forceinline__ RawPiece<XT, CW, CODES> raw_piece(const RowSumTask& K, int64_t row, int64_t col, bool full) {
  typedef typename Elem<XT>::T T;
  RawPiece<XT, CW, CODES> o;
  if constexpr (CODES) {
    const uint8_t* p = static_cast<const uint8_t*>(K.src) + row * K.ld + col;
    o.e = K.exps[row * (K.ld / kAct8Block) + col / kAct8Block];
    if constexpr (CW == 8) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      o.d[0] = v.x;
      o.d[1] = v.y;
    } else {
      o.d[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  } else {
    constexpr int kWords = ColPiece<XT, CW>::kWords;
    const T* p = static_cast<const T*>(K.src) + row * K.ld + col;
    if (full) {
      if constexpr (kWords == 4) {
        const u32x4 v = load16_any(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) o.d[i] = v[i];
      } else {
        const u32x2_any v = *reinterpret_cast<const u32x2_any*>(p);
        o.d[0] = v.x;
        o.d[1] = v.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (XT == RQ_DTYPE_F32) {
          o.d[i] = col + i < K.C ? f2u(p[i]) : 0u;
        } else {
          o.d[i] = (col + 2 * i < K.C ? uint32_t(p[2 * i]) : 0u) |
                   (col + 2 * i + 1 < K.C ? uint32_t(p[2 * i + 1]) << 16 : 0u);
        }
      }
    }
  }
  return o;
}

template <int XT, int CW, bool CODES>
__device__ __forceinline__ ColPiece<XT, CW> col_piece(const RawPiece<XT, CW, CODES>& r) {
  ColPiece<XT, CW> o;
  if constexpr (!CODES) {
#pragma unroll
    for (int i = 0; i < ColPiece<XT, CW>::kWords; ++i) o.d[i] = r.d[i];
  } else {
#pragma unroll
    for (int i = 0; i < CW / 4; ++i) {
      if constexpr (XT == RQ_DTYPE_F32) {
        o.d[4 * i] = f2u(act8_value<0>(r.d[i], int(r.e)));
        o.d[4 * i + 1] = f2u(act8_value<1>(r.d[i], int(r.e)));
        o.d[4 * i + 2] = f2u(act8_value<2>(r.d[i], int(r.e)));
        o.d[4 * i + 3] = f2u(act8_value<3>(r.d[i], int(r.e)));
      } else {
        const u32x2 v = act8_pairs<XT>(r.d[i], int(r.e));
        o.d[2 * i] = v.x;
        o.d[2 * i + 1] = v.y;
      }
    }
  }
  return o;
}

struct RowSumChunk {
  int adapter, t0, slot;
  int64_t live;  // slots from the first of tile t0 on
};

template <int XT, int JB, bool CODES>
__device__ __forceinline__ void rowsum_body(const RowSumArgs& a, const RowSumTask& K, const RowSumChunk& ch, int64_t c0, int j0,
                                            float (*red)[16 * rowsum_cw<XT>(JB)][16 * JB + 1]) {
  typedef typename Elem<XT>::T T;
  constexpr int CW = rowsum_cw<XT>(JB);
  constexpr int kWords = ColPiece<XT, CW>::kWords;
  constexpr int kPlanes = XT == RQ_DTYPE_F32 ? 1 : 2;
  constexpr int kOps = XT == RQ_DTYPE_F32 ? 2 : 1;  // 16-byte operands of eight slots
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t col = c0 + CW * i16;
  const bool full = c0 + 16 * CW <= K.C;            // all columns
  const int64_t lcol = full || col < K.C ? col : 0;  // lanes past the end repeat column 0: their sums are not stored
  const int64_t base = int64_t(kTileRows) * ch.t0;
  const T* opt = static_cast<const T*>(K.opt) + opt_at<XT>(base + 8 * g, i16, a.rp);

  f32x4 acc[CW][JB];
#pragma unroll
  for (int c = 0; c < CW; ++c)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  typedef RawPiece<XT, CW, CODES> Raw;
  struct Ops {
    u32x4 u[JB][kPlanes][kOps];
  };
  auto rows_of = [&](int (&r)[8], int64_t s) {  // slots base + s + 8 g ..; past the last: -1
    if (a.rows.p) {
      const int32_t* p = a.rows.p + a.rows.off_rows() + base + s + 8 * g;
      const u32x4 lo = *reinterpret_cast<const u32x4*>(p), hi = *reinterpret_cast<const u32x4*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[e] = int(lo[e]);
        r[4 + e] = int(hi[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t m = base + s + 8 * g + e;
        r[e] = m < a.rows.M ? int(m) : -1;
      }
    }
  };
  auto load = [&](Raw (&raw)[8], const int (&r)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) raw[e] = raw_piece<XT, CW, CODES>(K, r[e] < 0 ? 0 : r[e], lcol, full || lcol + CW <= K.C);
  };
  auto operands = [&](Ops& o, int64_t s) {
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int p = 0; p < kPlanes; ++p)
#pragma unroll
        for (int k = 0; k < kOps; ++k)
          o.u[j][p][k] = *reinterpret_cast<const u32x4*>(opt + opt_at<XT>(s, rowsum_rank(j0, j, a.rp), a.rp) + 512 * p + 256 * k);
  };
  auto products = [&](const Raw (&raw)[8], const Ops& o, const int (&r)[8], bool last) {
    ColPiece<XT, CW> row[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) row[e] = col_piece<XT, CW, CODES>(raw[e]);
    if (last) {  // rows past the last count as zero
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int d = 0; d < kWords; ++d) row[e].d[d] = r[e] < 0 ? 0u : row[e].d[d];
    }
    if constexpr (XT == RQ_DTYPE_F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int c = 0; c < CW; ++c)
#pragma unroll
          for (int j = 0; j < JB; ++j) {
            const float x = u2f(row[e].d[c]), u = u2f(o.u[j][0][e >> 2][e & 3]);
            acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, u, acc[c][j], 0, 0, 0);
          }
    } else {
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        u32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[e] = __builtin_amdgcn_perm(row[2 * e + 1].d[c >> 1], row[2 * e].d[c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int p = 0; p < kPlanes; ++p)
#pragma unroll
          for (int j = 0; j < JB; ++j)
            acc[c][j] = p == 0 ? mma<XT>(x, o.u[j][p][0], acc[c][j]) : mma_lo<XT>(x, o.u[j][p][0], acc[c][j]);
      }
    }
  };
  // the next step's rows are known before its values are asked for; two or three waves a SIMD
  // with eight loads each cover more latency than fewer waves with two steps in flight
  const int64_t live = ch.live;
  constexpr int64_t kAhead = 32 * kMlWaves;
  int64_t s = 32 * wave;
  int r0[8], r1[8];
  if (s < live) rows_of(r0, s);
  for (; s < live; s += kAhead) {
    Raw x[8];
    Ops o;
    load(x, r0);
    operands(o, s);
    if (s + kAhead < live) rows_of(r1, s + kAhead);
    products(x, o, r0, s + 32 > live);
#pragma unroll
    for (int e = 0; e < 8; ++e) r0[e] = r1[e];
  }
  // register q of lane (i, g): column CW (4 g + q) + c, rank i
#pragma unroll
  for (int ph = 0; ph < 2; ++ph) {
    if ((wave >> 1) == 1 - ph) {
#pragma unroll
      for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int j = 0; j < JB; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float& v = red[wave & 1][CW * (4 * g + q) + c][16 * j + i16];
            v = ph == 0 ? acc[c][j][q] : __fadd_rn(acc[c][j][q], v);
          }
    }
    __syncthreads();
  }
  const int cols = int(std::min<int64_t>(K.C - c0, 16 * CW)), ranks = std::min(a.r - j0, 16 * JB);
  float* part = ch.slot >= 0 ? a.part + ch.slot * a.part_size + K.part_off : nullptr;
  T* out = static_cast<T*>(K.out) + ch.adapter * K.C * a.r;
  const float scale = live > 0 ? a.scaling[ch.adapter] : 0.0f;  // an adapter without rows: zeros, whatever its scaling
  for (int i = threadIdx.x; i < cols * ranks; i += kMlThreads) {
    const int c = K.rank_major ? i % cols : i / ranks, j = K.rank_major ? i / cols : i % ranks;
    const float v = live > 0 ? __fmul_rn(scale, __fadd_rn(red[0][c][j], red[1][c][j])) : 0.0f;
    const int64_t to = K.rank_major ? int64_t(j0 + j) * K.C + c0 + c : (c0 + c) * a.r + j0 + j;
    if (part) part[to] = v;
    else out[to] = from_f32<XT>(v);
  }
}

// (fp16's lo parts meet in registers of their own: 170 with 64 ranks a wave, two waves a SIMD unless
// three are asked for; a backward pass of 4096 rows, K 4096, N 14336, r 64: 108 us with two, 98 - 100
// with three.)
template <int XT, int JB>
__global__ __launch_bounds__(kMlThreads) __attribute__((amdgpu_waves_per_eu(XT == RQ_DTYPE_F16 && JB == 4 ? 3 : 2))) void rowsum_kernel(RowSumArgs a) {
  constexpr int kCols = 16 * rowsum_cw<XT>(JB);
  __shared__ float red[2][kCols][16 * JB + 1];
  RowSumChunk ch{0, 0, -1, 0};
  int t1;
  if (a.rows.p) {
    if (int(blockIdx.y) >= a.rows.p[1 + a.table]) return;
    const int32_t* c = a.rows.p + a.rows.off_chunks() + 4 * (int64_t(a.rows.C) * a.table + blockIdx.y);
    ch.adapter = c[0];
    ch.t0 = c[1];
    t1 = c[2];
    ch.slot = c[3];
  } else {
    const Chunks c = adapter_chunks(a.rows.T, a.rows.T, a.table);
    if (int(blockIdx.y) >= c.n) return;
    ch.t0 = c.tiles * int(blockIdx.y);
    t1 = ch.t0 + c.tiles < a.rows.T ? ch.t0 + c.tiles : a.rows.T;
    if (c.n > 1) ch.slot = int(blockIdx.y);
  }
  // all tiles of an adapter but its last are full
  if (t1 > ch.t0) ch.live = int64_t(kTileRows) * (t1 - 1 - ch.t0) + plan_tile(a.rows, t1 - 1).count;
  const int which = int(blockIdx.x) >= a.t[0].tiles ? 1 : 0;
  const RowSumTask& K = a.t[which];
  const int64_t c0 = int64_t(int(blockIdx.x) - (which ? a.t[0].tiles : 0)) * kCols;
  const int j0 = 16 * JB * int(blockIdx.z);
  if (K.exps) rowsum_body<XT, JB, true>(a, K, ch, c0, j0, red);
  else rowsum_body<XT, JB, false>(a, K, ch, c0, j0, red);
}

// Adapters of several chunks: their partial sums in order.
template <int XT>
__global__ __launch_bounds__(kMlThreads) void rowsum_finish_kernel(RowSumArgs a) {
  typedef typename Elem<XT>::T T;
  const int adapter = int(blockIdx.y);
  int chunks, first = 0;
  if (a.rows.p) {
    const int32_t* p = a.rows.p + a.rows.off_part() + 2 * (int64_t(a.rows.n) * a.table + adapter);
    chunks = p[0];
    first = p[1];
  } else {
    chunks = adapter_chunks(a.rows.T, a.rows.T, a.table).n;
  }
  if (chunks == 1) return;
  for (int w = 0; w < a.n; ++w) {
    const RowSumTask& K = a.t[w];
    const int64_t n = K.C * a.r;
    T* out = static_cast<T*>(K.out) + adapter * n;
    const float* part = a.part + first * a.part_size + K.part_off;
    for (int64_t i = int64_t(blockIdx.x) * kMlThreads + threadIdx.x; i < n; i += int64_t(gridDim.x) * kMlThreads) {
      float v = 0.0f;
#pragma unroll 4
      for (int s = 0; s < chunks; ++s) v = __fadd_rn(v, part[s * a.part_size + i]);
      out[i] = from_f32<XT>(v);
    }
  }
}

// The table of chunks: the coarser one where its sums cannot meet in a second launch, or
// where its workgroups fill the GPU (4096 rows, K + N 18432, r 64: backward 97 us coarse,
// 123 fine, whose partial sums are four times as many).
int rowsum_table(const RowsPlan& rows, int64_t cols, int wg_cols, int cus) {
  const int64_t tiles = ceil_div(cols, wg_cols);
  return rows.T <= chunk_least(1) || tiles * ceil_div(ceil_div(rows.M, kTileRows), chunk_least(1)) >= cus ? 1 : 0;
}

// Partial slots that `table` may take.
int64_t rowsum_parts(const RowsPlan& rows, int table) {
  if (rows.p) return rows.T > chunk_least(table) ? std::min<int64_t>(kMaxParts, 2 * ceil_div(rows.T, chunk_least(table))) : 0;
  const int64_t c = adapter_chunks(rows.T, rows.T, table).n;
  return c > 1 ? c : 0;
}

template <int XT>
int run_rowsum(RowSumArgs a, hipStream_t stream) {
  const int jb = rowsum_blocks(a.rp);
  int tiles = 0;
  int64_t most = 0;
  for (int i = 0; i < a.n; ++i) {
    a.t[i].tiles = int(ceil_div(a.t[i].C, 16 * rowsum_cw<XT>(jb)));
    tiles += a.t[i].tiles;
    most = std::max(most, a.t[i].C * a.r);
  }
  if (a.rows.C > 65535) return RQ_ERR_UNSUPPORTED;
  const dim3 grid(unsigned(tiles), unsigned(a.rows.C), unsigned(ceil_div(a.rp, 16 * jb)));
  if (jb == 1) rowsum_kernel<XT, 1><<<grid, kMlThreads, 0, stream>>>(a);
  else if (jb == 2) rowsum_kernel<XT, 2><<<grid, kMlThreads, 0, stream>>>(a);
  else rowsum_kernel<XT, 4><<<grid, kMlThreads, 0, stream>>>(a);
  const int st = rq_check_launch();
  if (st != RQ_OK || rowsum_parts(a.rows, a.table) == 0) return st;
  const dim3 fgrid(unsigned(std::min<int64_t>(ceil_div(most, kMlThreads), std::max<int64_t>(4096 / a.rows.n, 64))), unsigned(a.rows.p ? a.rows.n : 1));
  rowsum_finish_kernel<XT><<<fgrid, kMlThreads, 0, stream>>>(a);
  return rq_check_launch();
}

namespace {

constexpr int64_t kMaxRank = 512;

size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

struct Sizes {
  int64_t M, K, N, n, r;
  int es;   // of an element
  int step;
};

int check_sizes(int dtype, int64_t M, int64_t K, int64_t N, int64_t n, int64_t r, Sizes* s) {
  if (!valid_float_dtype(dtype)) return RQ_ERR_BAD_DTYPE;
  if (M < 0 || K < 1 || N < 1 || n < 1 || r < 1) return RQ_ERR_BAD_SHAPE;
  if (M > (int64_t(1) << 30) || K > INT32_MAX || N > INT32_MAX || n > kMaxAdapters || r > kMaxRank) return RQ_ERR_UNSUPPORTED;
  *s = Sizes{M, K, N, n, r, int(dtype_size(dtype)), dtype == RQ_DTYPE_F32 ? 16 : 32};
  return RQ_OK;
}

struct ForwardPlan {
  int splits;
  int64_t per;
  size_t bytes;  // the splits' sums
};

ForwardPlan plan_forward(const Sizes& s, const RowsPlan& rows) {
  ForwardPlan p{};
  plan_shrink(rows.T, s.K, s.step, device_cus(), &p.splits, &p.per);
  p.bytes = up256(size_t(p.splits) * rows.slots() * rank_pad(s.r) * 4);
  return p;
}

struct BackwardPlan {
  int splits, table;
  int64_t per;
  size_t part, gt, sums, bytes;
  int64_t part_size;
};

BackwardPlan plan_backward(const Sizes& s, const RowsPlan& rows) {
  BackwardPlan p{};
  const int64_t rp = rank_pad(s.r), slots = rows.slots();
  const int cus = device_cus(), jb = rowsum_blocks(int(rp));
  plan_shrink(rows.T, s.N, s.step, cus, &p.splits, &p.per);
  p.table = rowsum_table(rows, s.K + s.N, 16 * (s.es == 4 ? rowsum_cw<RQ_DTYPE_F32>(jb) : rowsum_cw<RQ_DTYPE_BF16>(jb)), cus);
  p.part_size = ceil_div((s.K + s.N) * s.r, 8) * 8;
  size_t off = 0;
  auto take = [&](size_t b) {
    const size_t o = off;
    off += up256(b);
    return o;
  };
  p.part = take(size_t(p.splits) * slots * rp * 4);
  p.gt = take(size_t(slots) * rp * 4);
  p.sums = take(size_t(rowsum_parts(rows, p.table)) * p.part_size * 4);
  p.bytes = off;
  return p;
}

struct ForwardCall {
  Sizes s;
  RowsPlan rows;
  const void* x;
  int64_t ldx;
  const void* a;
  const void* b;
  const float* scaling;
  const void* base;
  int64_t ld_base;
  void* out;
  int64_t ld_out;
  void* u;
};

template <int XT>
int forward(const ForwardCall& c, char* ws, hipStream_t stream) {
  const ForwardPlan p = plan_forward(c.s, c.rows);
  const int r = int(c.s.r), rp = int(rank_pad(c.s.r));
  float* part = reinterpret_cast<float*>(ws);
  const ShrinkArgs sh{c.rows, c.x, c.ldx, c.s.K, c.a, c.s.r * c.s.K, r, rp, p.splits, p.per, part};
  const int st = run_shrink<XT, false>(sh, stream);
  if (st != RQ_OK) return st;
  const ExpandArgs e{c.rows, part, p.splits, r, rp, c.b, c.s.N * c.s.r, c.s.N, c.scaling, c.base, c.ld_base, c.out, c.ld_out,
                     c.u, 0, 0};
  return run_expand<XT, true>(e, device_cus(), stream);
}

struct BackwardCall {
  Sizes s;
  RowsPlan rows;
  const void* x;        // rows, or codes
  const uint8_t* exps;  // of codes
  int64_t ldx;
  const void* dy;
  int64_t lddy;
  const void* a;
  const void* b;
  const float* scaling;
  const void* u;
  const void* dx_base;
  int64_t ld_dx_base;
  void* dx;
  int64_t lddx;
  void* da;
  void* db;
};

template <int XT>
int backward(const BackwardCall& c, char* ws, hipStream_t stream) {
  const BackwardPlan p = plan_backward(c.s, c.rows);
  const int r = int(c.s.r), rp = int(rank_pad(c.s.r));
  float* part = reinterpret_cast<float*>(ws + p.part);
  int st = RQ_OK;
  if (c.dx || c.da) {
    const ShrinkArgs sh{c.rows, c.dy, c.lddy, c.s.N, c.b, c.s.N * c.s.r, r, rp, p.splits, p.per, part};
    if ((st = run_shrink<XT, true>(sh, stream)) != RQ_OK) return st;
  }
  void* gt = c.da ? ws + p.gt : nullptr;
  if (c.dx) {
    const ExpandArgs e{c.rows, part, p.splits, r, rp, c.a, c.s.r * c.s.K, c.s.K, c.scaling, c.dx_base, c.ld_dx_base, c.dx, c.lddx,
                       gt, 0, 0};
    st = run_expand<XT, false>(e, device_cus(), stream);
  } else if (c.da) {
    st = run_operands<XT>(OperandsArgs{c.rows, r, rp, part, p.splits, gt}, stream);
  }
  if (st != RQ_OK) return st;
  RowSumArgs q{};
  q.rows = c.rows;
  q.table = p.table;
  q.r = r;
  q.rp = rp;
  q.scaling = c.scaling;
  q.part = reinterpret_cast<float*>(ws + p.sums);
  q.part_size = p.part_size;
  if (c.db) q.t[q.n++] = RowSumTask{c.dy, nullptr, c.lddy, c.s.N, c.u, c.db, false, 0, 0};
  if (c.da) q.t[q.n++] = RowSumTask{c.x, c.exps, c.ldx, c.s.K, gt, c.da, true, c.s.N * c.s.r, 0};
  return q.n > 0 ? run_rowsum<XT>(q, stream) : RQ_OK;
}

// Rows of the plan given, or of one adapter.
int check_rows(const void* plan, int64_t plan_bytes, const Sizes& s, RowsPlan* rows) {
  if (!plan && s.n != 1) return RQ_ERR_NULL_POINTER;
  *rows = rows_plan(static_cast<const int32_t*>(plan), s.M, s.n);
  if (plan && plan_bytes < 4 * rows->words()) return RQ_ERR_BAD_SHAPE;
  return plan && !aligned(plan, 16) ? RQ_ERR_BAD_ALIGNMENT : RQ_OK;
}

}  // namespace
}  // namespace rq

extern "C" int rq_multi_lora_u_size(int64_t M, int64_t n, int64_t rank, int grouped, int64_t* bytes) {
  using namespace rq;
  if (!bytes) return RQ_ERR_NULL_POINTER;
  if (M < 0 || n < 1 || rank < 1 || M > (int64_t(1) << 30)) return RQ_ERR_BAD_SHAPE;
  if (n > kMaxAdapters || rank > kMaxRank) return RQ_ERR_UNSUPPORTED;
  static const int32_t some = 0;
  *bytes = rows_plan(grouped ? &some : nullptr, M, n).slots() * rank_pad(rank) * 4;
  return RQ_OK;
}

extern "C" int rq_multi_lora_scratch_size(int dtype, int64_t M, int64_t K, int64_t N, int64_t n, int64_t rank, int grouped,
                                          int backward, int64_t* bytes) {
  using namespace rq;
  if (!bytes) return RQ_ERR_NULL_POINTER;
  Sizes s{};
  const int st = check_sizes(dtype, M, K, N, n, rank, &s);
  if (st != RQ_OK) return st;
  static const int32_t some = 0;
  const RowsPlan rows = rows_plan(grouped ? &some : nullptr, M, n);
  *bytes = int64_t(backward ? plan_backward(s, rows).bytes : plan_forward(s, rows).bytes);
  return RQ_OK;
}

extern "C" int rq_multi_lora(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* plan,
                             int64_t plan_bytes, const void* lora_a, const void* lora_b, const float* scaling, int64_t n,
                             int64_t rank, int64_t N, const void* base, int64_t ld_base, void* out, int64_t ld_out,
                             void* u, void* scratch, int64_t scratch_bytes, hipStream_t stream) {
  using namespace rq;
  ForwardCall c{};
  int st = check_sizes(dtype, M, K, N, n, rank, &c.s);
  if (st != RQ_OK) return st;
  if (ldx < K || ld_out < N || (base && ld_base < N)) return RQ_ERR_BAD_SHAPE;
  if (M == 0) return RQ_OK;
  if (!x || !lora_a || !lora_b || !scaling || !out || !scratch) return RQ_ERR_NULL_POINTER;
  if ((st = check_rows(plan, plan_bytes, c.s, &c.rows)) != RQ_OK) return st;
  if (!aligned(x, c.s.es) || !aligned(lora_a, c.s.es) || !aligned(lora_b, c.s.es) || !aligned(out, c.s.es) ||
      (base && !aligned(base, c.s.es)) || !aligned(scratch, 256) || !aligned(scaling, 4) || (u && !aligned(u, 16)))
    return RQ_ERR_BAD_ALIGNMENT;
  if (scratch_bytes < int64_t(plan_forward(c.s, c.rows).bytes)) return RQ_ERR_WORKSPACE;
  c.x = x;
  c.ldx = ldx;
  c.a = lora_a;
  c.b = lora_b;
  c.scaling = scaling;
  c.base = base;
  c.ld_base = ld_base;
  c.out = out;
  c.ld_out = ld_out;
  c.u = u;
  RQ_DISPATCH_DT(dtype, XT, return forward<XT>(c, static_cast<char*>(scratch), stream));
  return RQ_OK;
}

extern "C" int rq_multi_lora_grads(const void* x, const uint8_t* x_exponents, int dtype, int64_t M, int64_t K, int64_t ldx,
                                   const void* dy, int64_t N, int64_t lddy, const void* plan, int64_t plan_bytes,
                                   const void* lora_a, const void* lora_b, const float* scaling, int64_t n, int64_t rank,
                                   const void* u, const void* dx_base, int64_t ld_dx_base, void* dx, int64_t lddx, void* da,
                                   void* db, void* scratch, int64_t scratch_bytes, hipStream_t stream) {
  using namespace rq;
  BackwardCall c{};
  int st = check_sizes(dtype, M, K, N, n, rank, &c.s);
  if (st != RQ_OK) return st;
  const int64_t pitch = ceil_div(K, kAct8Block) * kAct8Block;
  if (lddy < N || (da && ldx < K) || (da && x_exponents && ldx != pitch) || (dx && lddx < K) || (dx && dx_base && ld_dx_base < K))
    return RQ_ERR_BAD_SHAPE;
  if (!dx && !da && !db) return RQ_OK;
  if (!dy || !lora_a || !lora_b || !scaling || !scratch || (da && !x) || (db && !u)) return RQ_ERR_NULL_POINTER;
  if (M == 0) return RQ_ERR_BAD_SHAPE;
  if ((st = check_rows(plan, plan_bytes, c.s, &c.rows)) != RQ_OK) return st;
  const int es = c.s.es;
  if (!aligned(dy, es) || !aligned(lora_a, es) || !aligned(lora_b, es) || (dx && !aligned(dx, es)) || (da && !aligned(da, es)) ||
      (db && !aligned(db, es)) || (dx_base && !aligned(dx_base, es)) || !aligned(scratch, 256) || !aligned(scaling, 4) ||
      (u && !aligned(u, 16)) || (da && !aligned(x, x_exponents ? 16 : es)))
    return RQ_ERR_BAD_ALIGNMENT;
  if (scratch_bytes < int64_t(plan_backward(c.s, c.rows).bytes)) return RQ_ERR_WORKSPACE;
  c.x = x;
  c.exps = x_exponents;
  c.ldx = ldx;
  c.dy = dy;
  c.lddy = lddy;
  c.a = lora_a;
  c.b = lora_b;
  c.scaling = scaling;
  c.u = u;
  c.dx_base = dx_base;
  c.ld_dx_base = ld_dx_base;
  c.dx = dx;
  c.lddx = lddx;
  c.da = da;
  c.db = db;
  RQ_DISPATCH_DT(dtype, XT, return backward<XT>(c, static_cast<char*>(scratch), stream));
  return RQ_OK;
}
