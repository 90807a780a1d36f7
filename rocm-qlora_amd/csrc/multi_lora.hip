// The adapters' products over grouped rows (rq_multi_lora.h).
//
// All of them are bound by memory: a row meets r <= 64 ranks, some 4 r operations a
// byte at most, a tenth of what the matrix cores do in the time the byte takes.
// So rows are loaded straight into operand registers, 16 bytes a lane, and the
// adapters' factors, which the tiles of an adapter share, come from the L2.
#include "rq_multi_lora.h"

#include "rq_act8.h"
#include "rq_launch.h"
#include "rq_linear_dev.h"

#include <algorithm>

namespace rq {

constexpr int kMlThreads = 256;
constexpr int kMlWaves = kMlThreads / 64;

// ---- shrink ---------------------------------------------------------------------
// A workgroup takes a tile's rows over a split of K; its four waves divide the split
// and meet in LDS.  A wave holds the tile's 16-row blocks (1 to 4, as many as the
// tile has) times JB blocks of 16 ranks, so that a factor's piece is loaded once
// for the tile.
template <int XT, int NRB, int JB>
__device__ __forceinline__ void shrink_body(const ShrinkArgs& a, const Tile& tile, int t, int split, int j0, float* red) {
  typedef typename Elem<XT>::T T;
  constexpr int V = Elem<XT>::kVec, kStep = Elem<XT>::kStep;
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t slot0 = int64_t(kTileRows) * t;
  const T* xr[NRB];
  const T* sr[JB];
  bool jlive[JB];
#pragma unroll
  for (int b = 0; b < NRB; ++b) {
    const int i = 16 * b + i16;
    // rows past the tile's last repeat its first: their sums are not read
    const int row = plan_row(a.rows, slot0 + (i < tile.count ? i : 0));
    xr[b] = static_cast<const T*>(a.x) + int64_t(row) * a.ldx + V * g;
  }
#pragma unroll
  for (int b = 0; b < JB; ++b) {
    const int j = j0 + 16 * b + i16;
    jlive[b] = j < a.r;
    sr[b] = static_cast<const T*>(a.s) + tile.adapter * a.s_adapter + int64_t(jlive[b] ? j : 0) * a.ld_s + V * g;
  }
  f32x4 acc[NRB][JB];
#pragma unroll
  for (int b = 0; b < NRB; ++b)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t per = a.k_per_split / kMlWaves;
  const int64_t kb = split * a.k_per_split + wave * per;
  const int64_t ke = std::min<int64_t>(kb + per, a.K);
  // whole steps, the next one's loads in flight over this one's products
  auto load = [&](u32x4 (&x)[NRB], u32x4 (&s)[JB], int64_t k) {
#pragma unroll
    for (int b = 0; b < NRB; ++b) x[b] = load16_any(xr[b] + k);
#pragma unroll
    for (int j = 0; j < JB; ++j) s[j] = load16_any(sr[j] + k);
  };
  auto products = [&](const u32x4 (&x)[NRB], const u32x4 (&s)[JB]) {
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      const u32x4 f = jlive[j] ? s[j] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int b = 0; b < NRB; ++b) acc[b][j] = mma<XT>(x[b], f, acc[b][j]);
    }
  };
  int64_t k = kb;
  if (k + kStep <= ke) {
    u32x4 x0[NRB], s0[JB], x1[NRB], s1[JB];
    load(x0, s0, k);
    for (;;) {
      const int64_t k1 = k + kStep, k2 = k1 + kStep;
      const bool more1 = k1 + kStep <= ke, more2 = k2 + kStep <= ke;
      if (more1) load(x1, s1, k1);
      products(x0, s0);
      k = k1;
      if (!more1) break;
      if (more2) load(x0, s0, k2);
      products(x1, s1);
      k = k2;
      if (!more2) break;
    }
  }
  if (k < ke) {  // the end of the rows
    u32x4 x[NRB], s[JB];
#pragma unroll
    for (int b = 0; b < NRB; ++b) x[b] = load16_part<XT>(xr[b] + k, ke - k - V * g);
#pragma unroll
    for (int j = 0; j < JB; ++j) s[j] = load16_part<XT>(sr[j] + k, ke - k - V * g);
    products(x, s);
  }
  // waves summed as (0 + 2) + (1 + 3); register q of lane (i, g) is row 4 g + q, rank i
  constexpr int kPitch = 16 * JB + 1;
  auto at = [&](int w, int b, int j, int q) -> float& {
    return red[(w * 16 * NRB + 16 * b + 4 * g + q) * kPitch + 16 * j + i16];
  };
  if (wave >= 2) {
#pragma unroll
    for (int b = 0; b < NRB; ++b)
#pragma unroll
      for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) at(wave - 2, b, j, q) = acc[b][j][q];
  }
  __syncthreads();
  if (wave < 2) {
#pragma unroll
    for (int b = 0; b < NRB; ++b)
#pragma unroll
      for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          acc[b][j][q] = __fadd_rn(acc[b][j][q], at(wave, b, j, q));
          if (wave == 1) at(1, b, j, q) = acc[b][j][q];
        }
  }
  __syncthreads();
  if (wave == 0) {
    float* out = a.part + (int64_t(split) * a.rows.slots() + slot0) * a.r16 + j0;
#pragma unroll
    for (int b = 0; b < NRB; ++b)
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        if (j0 + 16 * j >= a.r16) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          out[int64_t(16 * b + 4 * g + q) * a.r16 + 16 * j + i16] = __fadd_rn(acc[b][j][q], at(1, b, j, q));
      }
  }
}

template <int XT, int JB>
__global__ __launch_bounds__(kMlThreads) void shrink_kernel(ShrinkArgs a) {
  __shared__ float red[2 * 64 * (16 * JB + 1)];
  const int t = int(blockIdx.x % unsigned(a.rows.T)), split = int(blockIdx.x / unsigned(a.rows.T));
  const int j0 = 16 * JB * int(blockIdx.y);
  const Tile tile = plan_tile(a.rows, t);
  if (tile.count == 0 || tile.adapter < 0) return;
  if (tile.count <= 16) shrink_body<XT, 1, JB>(a, tile, t, split, j0, red);
  else if (tile.count <= 32) shrink_body<XT, 2, JB>(a, tile, t, split, j0, red);
  else shrink_body<XT, 4, JB>(a, tile, t, split, j0, red);
}

// About four workgroups a compute unit, each wave with at least four steps.
void plan_shrink(int64_t T, int64_t K, int step, int cus, int* splits, int64_t* per) {
  const int64_t unit = int64_t(step) * kMlWaves;
  int64_t s = ceil_div(4 * cus, std::max<int64_t>(T, 1));
  s = std::min(s, std::max<int64_t>(K / (4 * unit), 1));
  s = std::min<int64_t>(std::max<int64_t>(s, 1), 16);
  *per = ceil_div(ceil_div(K, s), unit) * unit;
  *splits = int(ceil_div(K, *per));
}

template <int XT>
int run_shrink(const ShrinkArgs& a, hipStream_t stream) {
  const int jb = a.r16 <= 16 ? 1 : (a.r16 <= 32 ? 2 : 4);
  if (int64_t(a.rows.T) * a.splits > kMaxThreads1D / kMlThreads) return RQ_ERR_UNSUPPORTED;
  const dim3 grid(unsigned(int64_t(a.rows.T) * a.splits), unsigned(ceil_div(a.r16, 16 * jb)));
  if (jb == 1) shrink_kernel<XT, 1><<<grid, kMlThreads, 0, stream>>>(a);
  else if (jb == 2) shrink_kernel<XT, 2><<<grid, kMlThreads, 0, stream>>>(a);
  else shrink_kernel<XT, 4><<<grid, kMlThreads, 0, stream>>>(a);
  return rq_check_launch();
}

// ---- finish ---------------------------------------------------------------------
// A thread takes eight slots of one rank.  Slots of a tile past its rows get zeros:
// the row sums read them.
template <int XT>
__global__ __launch_bounds__(kMlThreads) void finish_kernel(FinishArgs a, unsigned per_job) {
  typedef typename Elem<XT>::T T;
  const int which = int(blockIdx.x / per_job);
  const FinishJob& J = a.job[which];
  const int64_t i = int64_t(blockIdx.x % per_job) * kMlThreads + threadIdx.x;
  const int64_t s8 = i / a.r16;
  const int j = int(i - s8 * a.r16);
  const int64_t slots = a.rows.slots(), s0 = 8 * s8;
  if (s0 >= slots) return;
  const int t = int(s0 / kTileRows);
  const Tile tile = plan_tile(a.rows, t);
  if (tile.count == 0 || tile.adapter < 0) return;
  const int live = tile.count - int(s0 - int64_t(kTileRows) * t);  // of these slots
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  for (int k = 0; k < J.splits; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < live) v[e] = __fadd_rn(v[e], J.part[(int64_t(k) * slots + s0 + e) * a.r16 + j]);
  }
  if (J.sum) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < live) J.sum[(s0 + e) * a.r16 + j] = v[e];
  }
  if (J.scaled) {
    const float s = a.scaling[tile.adapter];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < live ? __fmul_rn(v[e], s) : 0.0f;
  }
  if constexpr (XT == RQ_DTYPE_F32) {
    if (J.op) {
#pragma unroll
      for (int e = 0; e < 8; ++e) static_cast<float*>(J.op)[(s0 + e) * a.r16 + j] = v[e];
    }
    if (J.opt) {
      f32x4* o = reinterpret_cast<f32x4*>(static_cast<float*>(J.opt) + int64_t(j) * slots + s0);
      o[0] = f32x4{v[0], v[1], v[2], v[3]};
      o[1] = f32x4{v[4], v[5], v[6], v[7]};
    }
  } else {
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = to_x16<XT>(v[e]);
      const float h = from_x16<XT>(hi[e]);
      // an infinity has no second part (inf - inf)
      lo[e] = to_x16<XT>(fabsf(h) == __builtin_inff() ? 0.0f : v[e] - h);
    }
    if (J.op) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        T* o = static_cast<T*>(J.op) + (s0 + e) * (2 * a.r16);
        o[j] = T(hi[e]);
        o[a.r16 + j] = T(lo[e]);
      }
    }
    if (J.opt) {
      T* o = static_cast<T*>(J.opt) + int64_t(j) * slots + s0;
      *reinterpret_cast<u32x4*>(o) =
          u32x4{hi[0] | hi[1] << 16, hi[2] | hi[3] << 16, hi[4] | hi[5] << 16, hi[6] | hi[7] << 16};
      *reinterpret_cast<u32x4*>(o + int64_t(a.r16) * slots) =
          u32x4{lo[0] | lo[1] << 16, lo[2] | lo[3] << 16, lo[4] | lo[5] << 16, lo[6] | lo[7] << 16};
    }
  }
}

template <int XT>
int run_finish(const FinishArgs& a, hipStream_t stream) {
  const int64_t per = ceil_div(a.rows.slots() / 8 * a.r16, kMlThreads);
  if (per * a.jobs > kMaxThreads1D / kMlThreads) return RQ_ERR_UNSUPPORTED;
  finish_kernel<XT><<<unsigned(per * a.jobs), kMlThreads, 0, stream>>>(a, unsigned(per));
  return rq_check_launch();
}

// ---- expand ---------------------------------------------------------------------
// A wave takes 16 kVec columns of half a tile (two 16-row blocks).  The factor is the
// A operand and the slots the B operand, so that a result register holds columns; the
// operand row i of product c is column kVec i + c, so that a lane ends with kVec
// adjacent columns for each of its four registers: whole 16-byte pieces of a row,
// 256 bytes of it by the four lane groups.
//
// The contraction runs over the hi ranks, then the lo ranks, 16 at a time in rank
// order: r16 is a multiple of 16, so a 32-rank step of 16-bit operands is two ranks
// blocks, hi and lo of the same 16 when r16 = 16.
// kVec ranks from `v` (of hi | lo) on for each of the kVec columns, lane group g at
// V g within the step
template <int XT, bool FACTOR_ROWS>
__device__ __forceinline__ void load_factor(u32x4 (&f)[Elem<XT>::kVec], const typename Elem<XT>::T* s, int64_t ld,
                                            int64_t C, int64_t col, int r, int j) {
  constexpr int V = Elem<XT>::kVec;
  const u32x4 zero = u32x4{0u, 0u, 0u, 0u};
  if constexpr (FACTOR_ROWS) {
    // column c's ranks j .. j + V - 1 are adjacent
#pragma unroll
    for (int c = 0; c < V; ++c)
      f[c] = col + c < C && j < r ? load16_part<XT>(s + (col + c) * ld + j, r - j) : zero;
  } else {
    // rank j + e's columns are adjacent: transpose V x V values
    u32x4 row[V];
#pragma unroll
    for (int e = 0; e < V; ++e) row[e] = j + e < r ? load16_part<XT>(s + (j + e) * ld + col, C - col) : zero;
    if constexpr (XT == RQ_DTYPE_F32) {
#pragma unroll
      for (int c = 0; c < V; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) f[c][e] = row[e][c];
    } else {
#pragma unroll
      for (int c = 0; c < V; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          f[c][e] = __builtin_amdgcn_perm(row[2 * e + 1][c >> 1], row[2 * e][c >> 1], c & 1 ? 0x07060302u : 0x05040100u);
    }
  }
}

constexpr int kExpandBlocks = 2;  // 16-row blocks of a workgroup

template <int XT, bool FACTOR_ROWS>
__global__ __launch_bounds__(kMlThreads) void expand_kernel(ExpandArgs a) {
  typedef typename Elem<XT>::T T;
  constexpr int V = Elem<XT>::kVec, kStep = Elem<XT>::kStep;
  constexpr int kParts = kTileRows / (16 * kExpandBlocks);
  const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = int(blockIdx.x % unsigned(a.chunks));
  const unsigned rest = blockIdx.x / unsigned(a.chunks);
  const int t = int(rest / kParts), part = int(rest % kParts);
  const Tile tile = plan_tile(a.rows, t);
  const int first = 16 * kExpandBlocks * part;
  if (first >= tile.count) return;
  if (tile.adapter < 0 && a.base == a.out && a.ld_base == a.ld_out) return;  // in place, nothing to add
  const int64_t c0 = (int64_t(chunk) * kMlWaves + wave) * (16 * V);
  if (c0 >= a.C) return;
  const int64_t slot0 = int64_t(kTileRows) * t + first;
  const int64_t col = c0 + V * i16;
  f32x4 acc[kExpandBlocks][V];
#pragma unroll
  for (int b = 0; b < kExpandBlocks; ++b)
#pragma unroll
    for (int c = 0; c < V; ++c) acc[b][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (tile.adapter >= 0) {
    const T* s = static_cast<const T*>(a.s) + tile.adapter * a.s_adapter;
    const int width = XT == RQ_DTYPE_F32 ? a.r16 : 2 * a.r16;
    const T* op = static_cast<const T*>(a.op) + slot0 * width;
    for (int v = 0; v < width; v += kStep) {
      const int at = v + V * g;
      const int j = at >= a.r16 ? at - a.r16 : at;
      u32x4 f[V];
      load_factor<XT, FACTOR_ROWS>(f, s, a.ld_s, a.C, col, a.r, j);
#pragma unroll
      for (int b = 0; b < kExpandBlocks; ++b) {
        if (first + 16 * b >= tile.count) break;
        const u32x4 u = *reinterpret_cast<const u32x4*>(op + int64_t(16 * b + i16) * width + at);
#pragma unroll
        for (int c = 0; c < V; ++c) acc[b][c] = mma<XT>(f[c], u, acc[b][c]);
      }
    }
  }
  const float scale = a.scaling && tile.adapter >= 0 ? a.scaling[tile.adapter] : 1.0f;
#pragma unroll
  for (int b = 0; b < kExpandBlocks; ++b) {
    const int i = first + 16 * b + i16;
    if (i >= tile.count) continue;
    const int64_t row = plan_row(a.rows, int64_t(kTileRows) * t + i);
    const T* base = static_cast<const T*>(a.base) + (a.base ? row * a.ld_base : 0);
    T* out = static_cast<T*>(a.out) + row * a.ld_out;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t c = c0 + V * (4 * g + q);
      if (c >= a.C) continue;
      float f[V];
      if (a.base) {
        unpack16<XT>(load16_part<XT>(base + c, a.C - c), f);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = 0.0f;
      }
      if (tile.adapter >= 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = __fadd_rn(f[e], __fmul_rn(scale, acc[b][e][q]));
      }
      store16_part<XT>(out + c, f, a.C - c);
    }
  }
}

template <int XT, bool FACTOR_ROWS>
int run_expand(ExpandArgs a, hipStream_t stream) {
  a.chunks = int(ceil_div(a.C, kMlWaves * expand_cols<XT>()));
  const int64_t blocks = int64_t(a.rows.T) * (kTileRows / (16 * kExpandBlocks)) * a.chunks;
  if (blocks > kMaxThreads1D / kMlThreads) return RQ_ERR_UNSUPPORTED;
  expand_kernel<XT, FACTOR_ROWS><<<unsigned(blocks), kMlThreads, 0, stream>>>(a);
  return rq_check_launch();
}

// ---- sums over the rows of an adapter ----------------------------------------------
// D[c][j] = sum_m x[row m][c] u[m][j], the contraction over the slow index of x: lane
// (i, g) loads CW columns of the eight rows of slots 8 g .. 8 g + 7, which byte permutes
// turn into CW operand rows of eight consecutive slots (16-bit; fp32 values are operands
// as they are).  A wave's step is 32 slots; the four waves take steps in turn and meet in
// LDS.  Each column tile of a chunk is a workgroup.
template <int XT, int CW>
struct ColPiece {
  uint32_t d[XT == RQ_DTYPE_F32 ? CW : CW / 2];
};

template <int XT, int CW>
__device__ __forceinline__ ColPiece<XT, CW> col_piece(const RowSumTask& T_, int64_t row, int64_t col) {
  typedef typename Elem<XT>::T T;
  constexpr int kWords = XT == RQ_DTYPE_F32 ? CW : CW / 2;
  ColPiece<XT, CW> o;
  if (T_.exps) {
    const uint8_t* p = static_cast<const uint8_t*>(T_.src) + row * T_.ld + col;
    const int e = T_.exps[row * (T_.ld / kAct8Block) + col / kAct8Block];
    uint32_t w[CW / 4];
    if constexpr (CW == 8) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      w[0] = v.x;
      w[1] = v.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < CW / 4; ++i) {
      if constexpr (XT == RQ_DTYPE_F32) {
        o.d[4 * i] = f2u(act8_value<0>(w[i], e));
        o.d[4 * i + 1] = f2u(act8_value<1>(w[i], e));
        o.d[4 * i + 2] = f2u(act8_value<2>(w[i], e));
        o.d[4 * i + 3] = f2u(act8_value<3>(w[i], e));
      } else {
        const u32x2 v = act8_pairs<XT>(w[i], e);
        o.d[2 * i] = v.x;
        o.d[2 * i + 1] = v.y;
      }
    }
    return o;
  }
  const T* p = static_cast<const T*>(T_.src) + row * T_.ld + col;
  if (col + CW <= T_.C) {
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
        o.d[i] = col + i < T_.C ? f2u(p[i]) : 0u;
      } else {
        o.d[i] = (col + 2 * i < T_.C ? uint32_t(p[2 * i]) : 0u) | (col + 2 * i + 1 < T_.C ? uint32_t(p[2 * i + 1]) << 16 : 0u);
      }
    }
  }
  return o;
}

template <int XT, int JB>
__global__ __launch_bounds__(kMlThreads) __attribute__((amdgpu_waves_per_eu(2))) void rowsum_kernel(RowSumArgs a) {
  typedef typename Elem<XT>::T T;
  constexpr int CW = rowsum_cw<XT>(JB), kCols = 16 * CW, kPitch = 16 * JB + 1;
  constexpr int kWords = XT == RQ_DTYPE_F32 ? CW : CW / 2;
  constexpr int kPlanes = XT == RQ_DTYPE_F32 ? 1 : 2;
  __shared__ float red[2][kCols][kPitch];
  const int tid = threadIdx.x, lane = tid & 63, i16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int adapter = 0, t0, t1, slot = -1;
  if (a.rows.p) {
    if (int(blockIdx.y) >= a.rows.p[1]) return;
    const int32_t* c = a.rows.p + a.rows.off_chunks() + 4 * int64_t(blockIdx.y);
    adapter = c[0];
    t0 = c[1];
    t1 = c[2];
    slot = c[3];
  } else {
    const int per = RowsPlan::chunk_tiles(a.rows.T);
    t0 = per * int(blockIdx.y);
    t1 = t0 + per < a.rows.T ? t0 + per : a.rows.T;
    if (a.rows.C > 1) slot = int(blockIdx.y);
  }
  const int which = int(blockIdx.x) >= a.t[0].tiles ? 1 : 0;
  const RowSumTask& K = a.t[which];
  const int64_t c0 = int64_t(int(blockIdx.x) - (which ? a.t[0].tiles : 0)) * kCols;
  const int j0 = 16 * JB * int(blockIdx.z);
  const int64_t col = c0 + CW * i16;
  const bool clive = col < K.C;
  const int64_t slots = a.rows.slots();

  f32x4 acc[CW][JB];
#pragma unroll
  for (int c = 0; c < CW; ++c)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int step = wave; step < 2 * (t1 - t0); step += kMlWaves) {
    const int t = t0 + (step >> 1);
    const Tile tile = plan_tile(a.rows, t);
    const int h = 32 * (step & 1);
    if (h >= tile.count) continue;
    const int64_t slot0 = int64_t(kTileRows) * t + h + 8 * g;
    ColPiece<XT, CW> row[8];
    // the loads first; rows past the tile's last repeat its first and count as zero
    const int64_t lcol = clive ? col : 0;
    int r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = plan_row(a.rows, h + 8 * g + e < tile.count ? slot0 + e : int64_t(kTileRows) * t);
#pragma unroll
    for (int e = 0; e < 8; ++e) row[e] = col_piece<XT, CW>(K, r[e], lcol);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int d = 0; d < kWords; ++d)
        if (!clive || h + 8 * g + e >= tile.count) row[e].d[d] = 0u;
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      if (j0 + 16 * j >= a.r16) continue;
      const T* u = static_cast<const T*>(K.opt) + int64_t(j0 + 16 * j + i16) * slots + slot0;
      if constexpr (XT == RQ_DTYPE_F32) {
        const f32x4 u0 = *reinterpret_cast<const f32x4*>(u), u1 = *reinterpret_cast<const f32x4*>(u + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int c = 0; c < CW; ++c)
            acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(row[e].d[c]), e < 4 ? u0[e & 3] : u1[e & 3], acc[c][j], 0, 0, 0);
      } else {
#pragma unroll
        for (int p = 0; p < kPlanes; ++p) {
          const u32x4 op = *reinterpret_cast<const u32x4*>(u + int64_t(p) * a.r16 * slots);
#pragma unroll
          for (int c = 0; c < CW; ++c) {
            u32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x[e] = __builtin_amdgcn_perm(row[2 * e + 1].d[c >> 1], row[2 * e].d[c >> 1],
                                           c & 1 ? 0x07060302u : 0x05040100u);
            acc[c][j] = mma<XT>(x, op, acc[c][j]);
          }
        }
      }
    }
  }
  // waves summed as (0 + 2) + (1 + 3); register q of lane (i, g) is column CW (4 g + q) + c, rank i
#pragma unroll
  for (int ph = 0; ph < 2; ++ph) {
    if ((wave >> 1) == 1 - ph) {
#pragma unroll
      for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int j = 0; j < JB; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float& o = red[wave & 1][CW * (4 * g + q) + c][16 * j + i16];
            o = ph == 0 ? acc[c][j][q] : __fadd_rn(acc[c][j][q], o);
          }
    }
    __syncthreads();
  }
  const int cols = int(std::min<int64_t>(K.C - c0, kCols)), ranks = std::min(a.r - j0, 16 * JB);
  for (int i = tid; i < cols * ranks; i += kMlThreads) {
    const int c = K.rank_major ? i % cols : i / ranks, j = K.rank_major ? i / cols : i % ranks;
    const float v = __fadd_rn(red[0][c][j], red[1][c][j]);
    const int64_t at = K.rank_major ? int64_t(j0 + j) * K.C + c0 + c : (c0 + c) * a.r + j0 + j;
    if (slot >= 0) a.part[slot * a.part_size + K.part_off + at] = v;
    else static_cast<T*>(K.out)[adapter * K.C * a.r + at] = from_f32<XT>(v);
  }
}

// Adapters of several chunks: their partial sums in order.  Adapters without rows:
// zeros.
template <int XT>
__global__ __launch_bounds__(kMlThreads) void rowsum_finish_kernel(RowSumArgs a) {
  typedef typename Elem<XT>::T T;
  const int adapter = int(blockIdx.y);
  int chunks = a.rows.C, first = 0;
  if (a.rows.p) {
    chunks = a.rows.p[a.rows.off_part() + 2 * int64_t(adapter)];
    first = a.rows.p[a.rows.off_part() + 2 * int64_t(adapter) + 1];
  }
  if (chunks == 1) return;
  for (int w = 0; w < a.n; ++w) {
    const RowSumTask& K = a.t[w];
    const int64_t n = K.C * a.r;
    T* out = static_cast<T*>(K.out) + adapter * n;
    for (int64_t i = int64_t(blockIdx.x) * kMlThreads + threadIdx.x; i < n; i += int64_t(gridDim.x) * kMlThreads) {
      float v = 0.0f;
      for (int s = 0; s < chunks; ++s) v = __fadd_rn(v, a.part[(first + s) * a.part_size + K.part_off + i]);
      out[i] = from_f32<XT>(v);
    }
  }
}

template <int XT>
int run_rowsum(RowSumArgs a, hipStream_t stream) {
  const int jb = a.r16 <= 16 ? 1 : (a.r16 <= 32 ? 2 : 4);
  int tiles = 0;
  int64_t most = 0;
  for (int i = 0; i < a.n; ++i) {
    a.t[i].tiles = int(ceil_div(a.t[i].C, 16 * rowsum_cw<XT>(jb)));
    tiles += a.t[i].tiles;
    most = std::max(most, a.t[i].C * a.r);
  }
  if (a.rows.C > 65535) return RQ_ERR_UNSUPPORTED;
  int st = RQ_OK;
  if (a.rows.C > 0) {
    const dim3 grid(unsigned(tiles), unsigned(a.rows.C), unsigned(ceil_div(a.r16, 16 * jb)));
    if (jb == 1) rowsum_kernel<XT, 1><<<grid, kMlThreads, 0, stream>>>(a);
    else if (jb == 2) rowsum_kernel<XT, 2><<<grid, kMlThreads, 0, stream>>>(a);
    else rowsum_kernel<XT, 4><<<grid, kMlThreads, 0, stream>>>(a);
    if ((st = rq_check_launch()) != RQ_OK) return st;
  }
  if (!a.rows.p && a.rows.C == 1) return RQ_OK;
  const dim3 grid(unsigned(std::min<int64_t>(ceil_div(most, kMlThreads), 1024)), unsigned(a.rows.p ? a.rows.n : 1));
  rowsum_finish_kernel<XT><<<grid, kMlThreads, 0, stream>>>(a);
  return rq_check_launch();
}

// ---- B [N, r] as rows of ranks [r16][ldt], for the backward's shrink --------------------
// A workgroup turns 256 rows of B of one adapter through LDS, if the adapter has rows.
constexpr int kTurnRows = 256, kTurnRanks = 16;

template <int XT>
__global__ __launch_bounds__(kMlThreads) void turn_kernel(RowsPlan rows, const void* b, int64_t N, int64_t ldb, int64_t b_adapter,
                                                          int r, int r16, void* bt, int64_t ldt) {
  typedef typename Elem<XT>::T T;
  __shared__ T tile[kTurnRanks][kTurnRows + 2];
  const int adapter = int(blockIdx.z), j0 = kTurnRanks * int(blockIdx.y);
  if (rows.p && rows.p[rows.off_part() + 2 * int64_t(adapter)] == 0) return;
  const int64_t n0 = int64_t(blockIdx.x) * kTurnRows;
  const T* src = static_cast<const T*>(b) + adapter * b_adapter;
  for (int i = threadIdx.x; i < kTurnRanks * kTurnRows; i += kMlThreads) {
    const int j = i % kTurnRanks, k = i / kTurnRanks;
    tile[j][k] = j0 + j < r && n0 + k < N ? src[(n0 + k) * ldb + j0 + j] : T(0);
  }
  __syncthreads();
  T* dst = static_cast<T*>(bt) + (int64_t(adapter) * r16 + j0) * ldt + n0;
  for (int i = threadIdx.x; i < kTurnRanks * kTurnRows; i += kMlThreads) {
    const int j = i / kTurnRows, k = i % kTurnRows;
    if (n0 + k < ldt) dst[j * ldt + k] = tile[j][k];
  }
}

template <int XT>
int run_turn(const RowsPlan& rows, const void* b, int64_t N, int64_t ldb, int64_t b_adapter, int r, int r16, void* bt,
             int64_t ldt, hipStream_t stream) {
  const dim3 grid(unsigned(ceil_div(ldt, kTurnRows)), unsigned(r16 / kTurnRanks), unsigned(rows.p ? rows.n : 1));
  turn_kernel<XT><<<grid, kMlThreads, 0, stream>>>(rows, b, N, ldb, b_adapter, r, r16, bt, ldt);
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

// widths of the finished operands of a slot: fp32, or hi | lo
size_t op_bytes(const Sizes& s, int64_t slots) { return size_t(slots) * rank16(s.r) * 4; }

struct ForwardPlan {
  int splits;
  int64_t per;
  size_t part, op, bytes;
};

ForwardPlan plan_forward(const Sizes& s, const RowsPlan& rows) {
  ForwardPlan p{};
  plan_shrink(rows.T, s.K, s.step, device_cus(), &p.splits, &p.per);
  p.part = 0;
  p.op = up256(size_t(p.splits) * rows.slots() * rank16(s.r) * 4);
  p.bytes = p.op + up256(op_bytes(s, rows.slots()));
  return p;
}

struct BackwardPlan {
  int splits;
  int64_t per, ldt;
  size_t bt, part, op, gt, ut, sums, bytes;
  int64_t part_size;
};

BackwardPlan plan_backward(const Sizes& s, const RowsPlan& rows) {
  BackwardPlan p{};
  const int64_t r16 = rank16(s.r), slots = rows.slots();
  plan_shrink(rows.T, s.N, s.step, device_cus(), &p.splits, &p.per);
  p.ldt = ceil_div(s.N, 8) * 8;
  p.part_size = (s.K + s.N) * s.r;
  size_t off = 0;
  auto take = [&](size_t b) {
    const size_t o = off;
    off += up256(b);
    return o;
  };
  p.bt = take(size_t(s.n) * r16 * p.ldt * s.es);
  p.part = take(size_t(p.splits) * slots * r16 * 4);
  p.op = take(op_bytes(s, slots));
  p.gt = take(op_bytes(s, slots));
  p.ut = take(op_bytes(s, slots));
  const int64_t parts = rows.p ? std::min<int64_t>(kMaxParts, 2 * ceil_div(rows.T, kChunkTiles)) : (rows.C > 1 ? rows.C : 0);
  p.sums = take(size_t(parts) * p.part_size * 4);
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
  float* u;
};

template <int XT>
int forward(const ForwardCall& c, char* ws, hipStream_t stream) {
  const ForwardPlan p = plan_forward(c.s, c.rows);
  const int r16 = int(rank16(c.s.r));
  ShrinkArgs sh{};
  sh.rows = c.rows;
  sh.x = c.x;
  sh.ldx = c.ldx;
  sh.K = c.s.K;
  sh.s = c.a;
  sh.ld_s = c.s.K;
  sh.s_adapter = c.s.r * c.s.K;
  sh.r = int(c.s.r);
  sh.r16 = r16;
  sh.splits = p.splits;
  sh.k_per_split = p.per;
  sh.part = reinterpret_cast<float*>(ws + p.part);
  int st = run_shrink<XT>(sh, stream);
  if (st != RQ_OK) return st;
  FinishArgs f{};
  f.rows = c.rows;
  f.r16 = r16;
  f.scaling = c.scaling;
  f.jobs = 1;
  f.job[0] = FinishJob{sh.part, p.splits, false, c.u, ws + p.op, nullptr};
  if ((st = run_finish<XT>(f, stream)) != RQ_OK) return st;
  ExpandArgs e{};
  e.rows = c.rows;
  e.op = ws + p.op;
  e.r = int(c.s.r);
  e.r16 = r16;
  e.s = c.b;
  e.s_adapter = c.s.N * c.s.r;
  e.ld_s = c.s.r;
  e.C = c.s.N;
  e.scaling = c.scaling;
  e.base = c.base;
  e.ld_base = c.ld_base;
  e.out = c.out;
  e.ld_out = c.ld_out;
  return run_expand<XT, true>(e, stream);
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
  const float* u;
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
  const int r16 = int(rank16(c.s.r));
  int st = RQ_OK;
  FinishArgs f{};
  f.rows = c.rows;
  f.r16 = r16;
  f.scaling = c.scaling;
  if (c.dx || c.da) {
    if ((st = run_turn<XT>(c.rows, c.b, c.s.N, c.s.r, c.s.N * c.s.r, int(c.s.r), r16, ws + p.bt, p.ldt, stream)) != RQ_OK) return st;
    ShrinkArgs sh{};
    sh.rows = c.rows;
    sh.x = c.dy;
    sh.ldx = c.lddy;
    sh.K = c.s.N;
    sh.s = ws + p.bt;
    sh.ld_s = p.ldt;
    sh.s_adapter = r16 * p.ldt;
    sh.r = int(c.s.r);
    sh.r16 = r16;
    sh.splits = p.splits;
    sh.k_per_split = p.per;
    sh.part = reinterpret_cast<float*>(ws + p.part);
    if ((st = run_shrink<XT>(sh, stream)) != RQ_OK) return st;
    f.job[f.jobs++] = FinishJob{sh.part, p.splits, true, nullptr, c.dx ? ws + p.op : nullptr, c.da ? ws + p.gt : nullptr};
  }
  if (c.db) f.job[f.jobs++] = FinishJob{c.u, 1, true, nullptr, nullptr, ws + p.ut};
  if (f.jobs == 0) return RQ_OK;
  if ((st = run_finish<XT>(f, stream)) != RQ_OK) return st;
  if (c.dx) {
    ExpandArgs e{};
    e.rows = c.rows;
    e.op = ws + p.op;
    e.r = int(c.s.r);
    e.r16 = r16;
    e.s = c.a;
    e.s_adapter = c.s.r * c.s.K;
    e.ld_s = c.s.K;
    e.C = c.s.K;
    e.base = c.dx_base;
    e.ld_base = c.ld_dx_base;
    e.out = c.dx;
    e.ld_out = c.lddx;
    if ((st = run_expand<XT, false>(e, stream)) != RQ_OK) return st;
  }
  RowSumArgs r{};
  r.rows = c.rows;
  r.r = int(c.s.r);
  r.r16 = r16;
  r.part = reinterpret_cast<float*>(ws + p.sums);
  r.part_size = p.part_size;
  if (c.db) r.t[r.n++] = RowSumTask{c.dy, nullptr, c.lddy, c.s.N, ws + p.ut, c.db, false, 0, 0};
  if (c.da) r.t[r.n++] = RowSumTask{c.x, c.exps, c.ldx, c.s.K, ws + p.gt, c.da, true, c.s.N * c.s.r, 0};
  return r.n > 0 ? run_rowsum<XT>(r, stream) : RQ_OK;
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

extern "C" int rq_multi_lora_slots(int64_t M, int64_t n, int grouped, int64_t* slots) {
  if (!slots) return RQ_ERR_NULL_POINTER;
  if (M < 0 || n < 1 || M > (int64_t(1) << 30)) return RQ_ERR_BAD_SHAPE;
  if (n > rq::kMaxAdapters) return RQ_ERR_UNSUPPORTED;
  static const int32_t some = 0;
  *slots = rq::rows_plan(grouped ? &some : nullptr, M, n).slots();
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
                             float* u, void* scratch, int64_t scratch_bytes, hipStream_t stream) {
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
                                   const float* u, const void* dx_base, int64_t ld_dx_base, void* dx, int64_t lddx, void* da,
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
