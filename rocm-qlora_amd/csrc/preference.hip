// Log-probabilities of labelled sequences, the preference loss on pairs of them,
// and the gradient of the logits.
//
//   lp[t] = z[t, y_t] - max z[t] - log sum_v exp(z[t, v] - max z[t]),  y_t = labels[t + 1]
//   L_i   = sum of lp over the labelled positions of sequence i (their mean if asked)
//   D_p   = beta ((L_p - R_p) - (L_{P+p} - R_{P+p}))
//   loss  = mean_p (1 - eps) softplus(-D_p) + eps softplus(D_p)
//   dz[t, v] = c_i ([v = y_t] - exp(z[t, v] - max z[t]) / sum),  c_i = d loss / d L_i
//
// Three launches.  The rows' maxima and sums are one pass over the labelled
// rows: every thread keeps its own running maximum m and the sum of 2^(x log2 e - n),
// n = ceil(m log2 e), which it rescales, by a power of two, when a piece of the row
// raises n; a row is split over workgroups when there are few.  With an integer n the
// argument is one fused multiply-add, rounded once and by 2^-24 of itself.
// The second launch joins the splits and sums each sequence, in fp64 and in a
// fixed order; the workgroup that ends last takes the pairs.  The gradient is a
// second pass: a pair's coefficient depends on every row of the pair.
// Bound by memory: the labelled rows read twice, every row of the gradient
// written once.  8336 rows of 128256 bf16 logits, 4862 of them labelled: sums 218 us
// (5.7 TB/s), gradient 635 (1.2 GB read, 2.1 written, 5.3 TB/s).  The sequences' launch is
// latency, 6.5 to 10 us.
#include "rq_io.h"
#include "rq_launch.h"
#include "rq_linear_dev.h"

#include <algorithm>

namespace rq {
namespace {

constexpr int kPfThreads = 256;
constexpr int kPfUnroll = 4;       // 16-byte loads of a thread in flight
constexpr int kPfSeqThreads = 1024;
constexpr float kLog2e = 1.44269504088896340736f;  // rounded to fp32

// Rows of logits: T of them, row t at z + (t / period) * outer + (t % period) * ld.
struct Rows {
  int64_t T, V, ld, period, outer;
  __device__ __forceinline__ int64_t at(int64_t t) const {
    return period ? (t / period) * outer + (t % period) * ld : t * ld;
  }
};

struct Labels {
  const int64_t* labels;   // [T]
  const int32_t* offsets;  // [S + 1], or nullptr: sequences of T / S rows
  int64_t S;
  int64_t ignore;
};

// The row's sequence (-1: none) and target: its label, -1 when it has none, -2 when
// the label is no index of the vocabulary (such a row counts as NaN).
struct RowTarget {
  int seq;
  int64_t target;
};

template <int NT>
__device__ __forceinline__ RowTarget row_target(const Labels& L, const Rows& r, int64_t t) {
  int64_t end;
  RowTarget o;
  if (L.offsets) {
    // offsets are ascending: the sequence is the number of starts up to t, less one
    int n = 0;
    for (int64_t i = threadIdx.x; i < ceil_div(L.S, NT) * NT; i += NT) n += __syncthreads_count(i < L.S && L.offsets[i] <= t);
    o.seq = n - 1;
    end = n > 0 ? int64_t(L.offsets[n]) : 0;
    if (t >= end) o.seq = -1;
  } else {
    const int64_t len = r.T / L.S;
    o.seq = int(t / len);
    end = (o.seq + 1) * len;
  }
  o.target = -1;
  if (o.seq >= 0 && t + 1 < end && t + 1 < r.T) {
    const int64_t y = L.labels[t + 1];
    if (y != L.ignore) o.target = y >= 0 && y < r.V ? y : -2;
  }
  return o;
}

// What the forward leaves for every row: its target (as above), sequence, maximum
// and sum (NaN for a row without a finite logit).
struct RowInfo {
  int32_t target;
  int32_t seq;
  float top;
  float sum;
};

// The largest maximum next to which terms count.  Their argument is off by the rounding of
// m log2 e, 64 at most: terms and sums stay within fp32, and the log-probability takes the same n.
// Past it fp32 values are 128 apart or more, and e^-128 is none.
constexpr float kHuge = 0x1p30f;
__device__ __forceinline__ bool huge(float m) { return !(fabsf(m) <= kHuge); }

// n of a maximum m, and a term of the sum relative to it.
__device__ __forceinline__ float base_of(float m) {
  return huge(m) ? (m > 0.0f ? 0x1p102f : -0x1p102f) : __builtin_ceilf(m * kLog2e);
}
__device__ __forceinline__ float term(float x, float n) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, -n)); }

// What a sum relative to m counts for relative to `top`, the largest of several: sides of a huge
// maximum count for nothing beside another one.
__device__ __forceinline__ float weight(float m, float top) {
  return m == top ? 1.0f : (huge(m) || huge(top)) ? 0.0f : __builtin_amdgcn_exp2f(base_of(m) - base_of(top));
}

// (m, s) joined with (m2, s2); an empty side has m = -inf, s = 0.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), f = weight(m, top), f2 = weight(m2, top);
  s = s * f + s2 * f2;  // a NaN on either side stays one
  m = top;
}

// The value of the lane that CTRL names, in the rows of 16 lanes that ROWS names (others: none).
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T from_lane(T v, T none) {
  constexpr int kWords = sizeof(T) / 4;
  struct Words {
    int w[kWords];
  };
  Words a = __builtin_bit_cast(Words, v), o = __builtin_bit_cast(Words, none);
#pragma unroll
  for (int i = 0; i < kWords; ++i) a.w[i] = __builtin_amdgcn_update_dpp(o.w[i], a.w[i], CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(T, a);
}

// op over the values of a wave's 64 lanes, for all of them: shifts by 1, 2, 4 and 8 within rows
// of 16 lanes, then the rows' last lanes.  Registers alone: with lane shuffles, which pass the
// LDS unit, and the sums joined in pairs the forward of 2084 rows of 32000 took 41.4 us for 39.0.
template <typename T, typename Op>
__device__ __forceinline__ T over_wave(T v, T none, Op op) {
  v = op(v, from_lane<0x111, 0xF>(v, none));
  v = op(v, from_lane<0x112, 0xF>(v, none));
  v = op(v, from_lane<0x114, 0xF>(v, none));
  v = op(v, from_lane<0x118, 0xF>(v, none));
  v = op(v, from_lane<0x142, 0xA>(v, none));
  v = op(v, from_lane<0x143, 0xC>(v, none));
  constexpr int kWords = sizeof(T) / 4;
  struct Words {
    int w[kWords];
  };
  Words a = __builtin_bit_cast(Words, v);
#pragma unroll
  for (int i = 0; i < kWords; ++i) a.w[i] = __builtin_amdgcn_readlane(a.w[i], 63);
  return __builtin_bit_cast(T, a);
}
__device__ __forceinline__ float wave_max(float v) {
  return over_wave(v, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); });
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
  return over_wave(v, T(0), [](T a, T b) { return a + b; });
}

// Piece [v0, v1) of a row that a workgroup takes: whole KiB but for the row's last.
template <int XT>
struct Piece {
  int64_t v0, v1;
};

template <int XT>
__device__ __forceinline__ Piece<XT> piece_of(int64_t V, int split, int splits) {
  constexpr int64_t W = Elem<XT>::kVec * 64;
  const int64_t per = ceil_div(ceil_div(V, splits), W) * W;
  const int64_t v0 = std::min<int64_t>(split * per, V);
  return Piece<XT>{v0, std::min<int64_t>(v0 + per, V)};
}

template <int XT>
__global__ __launch_bounds__(kPfThreads) void row_sums_kernel(Rows r, Labels L, const void* z, int splits, RowInfo* info,
                                                              float* part, uint32_t* done) {
  typedef typename Elem<XT>::T T;
  constexpr int VW = Elem<XT>::kVec;
  const int64_t t = blockIdx.x / unsigned(splits);
  const int split = int(blockIdx.x % unsigned(splits));
  if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0;
  const RowTarget rt = row_target<kPfThreads>(L, r, t);
  if (split == 0 && threadIdx.x == 0) {
    info[t].target = int32_t(rt.target);
    info[t].seq = rt.seq;
  }
  if (rt.target < 0) return;
  const T* row = static_cast<const T*>(z) + r.at(t);
  const Piece<XT> p = piece_of<XT>(r.V, split, splits);
  float m = -__builtin_inff(), s = 0.0f;
  float base = base_of(m);
  auto take = [&](const float* f, int count) {
    float top = m;
#pragma unroll
    for (int i = 0; i < count; ++i) top = fmaxf(top, f[i]);
    if (huge(top)) {  // -inf so far, or one that only its equals stand beside; a NaN still has to show
      if (top != m && !(s != s)) s = 0.0f;
#pragma unroll
      for (int i = 0; i < count; ++i) s += f[i] != f[i] ? f[i] : (f[i] == top && top > -__builtin_inff() ? 1.0f : 0.0f);
      m = top;
      base = base_of(top);
      return;
    }
    if (top > m) {
      const float n = base_of(top);
      // what a huge negative maximum or none left behind counts for nothing (but a NaN)
      s = huge(m) ? (s != s ? s : 0.0f) : s * __builtin_amdgcn_exp2f(base - n);
      base = n;
      m = top;
    }
#pragma unroll
    for (int i = 0; i < count; ++i) s += term(f[i], base);
  };
  constexpr int64_t kSpan = int64_t(kPfThreads) * VW;
  int64_t v = p.v0 + threadIdx.x * VW;
  for (; v + (kPfUnroll - 1) * kSpan + VW <= p.v1; v += kPfUnroll * kSpan) {
    u32x4 raw[kPfUnroll];
#pragma unroll
    for (int u = 0; u < kPfUnroll; ++u) raw[u] = load16_any(row + v + u * kSpan);
#pragma unroll
    for (int u = 0; u < kPfUnroll; ++u) {
      float f[VW];
      unpack16<XT>(raw[u], f);
      take(f, VW);
    }
  }
  for (; v < p.v1; v += kSpan) {
    if (v + VW <= p.v1) {
      float f[VW];
      unpack16<XT>(load16_any(row + v), f);
      take(f, VW);
    } else {
      for (int64_t i = v; i < p.v1; ++i) {
        const float f = to_f32<XT>(row[i]);
        take(&f, 1);
      }
    }
  }
  const float top = wave_max(m);
  s = wave_sum(s * weight(m, top));  // a NaN stays one
  m = top;
  __shared__ float wm[kPfThreads / 64], wsum[kPfThreads / 64];
  if ((threadIdx.x & 63) == 0) {
    wm[threadIdx.x >> 6] = m;
    wsum[threadIdx.x >> 6] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kPfThreads / 64; ++w) join(m, s, wm[w], wsum[w]);
    if (m == __builtin_inff()) s = __builtin_nanf("");
    part[2 * (t * splits + split)] = m;
    part[2 * (t * splits + split) + 1] = s;
  }
}

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

struct Pairs {
  const float* ref;  // [S] or nullptr: zeros
  float beta, eps;
  bool average;
  bool pairs;        // false: log-probabilities alone
};

// A workgroup per sequence: the sum of its rows' log-probabilities.  The last
// workgroup to end takes the pairs: sums[i] and counts[i] of the others are read
// past the L2 of its XCD, as they were written.
template <int XT>
__global__ __launch_bounds__(kPfSeqThreads) void sequences_kernel(Rows r, Labels L, const void* z, int splits, RowInfo* info,
                                                                  const float* part, uint32_t* done, double* sums,
                                                                  Pairs P, float* logps, float* loss, float* coef) {
  typedef typename Elem<XT>::T T;
  const int64_t i = blockIdx.x;
  int64_t b, e;
  if (L.offsets) {
    b = std::min<int64_t>(std::max<int64_t>(L.offsets[i], 0), r.T);
    e = std::min<int64_t>(std::max<int64_t>(L.offsets[i + 1], b), r.T);
  } else {
    b = i * (r.T / L.S);
    e = b + r.T / L.S;
  }
  double sum = 0.0;
  int count = 0;
  for (int64_t t = b + threadIdx.x; t < e; t += kPfSeqThreads) {
    const int y = info[t].target;
    if (y == -1 || info[t].seq != i) continue;
    ++count;
    float m = -__builtin_inff(), s = 0.0f;
    if (y >= 0) {
      for (int k = 0; k < splits; ++k) join(m, s, part[2 * (t * splits + k)], part[2 * (t * splits + k) + 1]);
      const float x = to_f32<XT>(static_cast<const T*>(z)[r.at(t) + y]);
      // log2 e as the sum's terms have it, so that its rounding is no error of x - m
      sum += huge(m) ? double(x) - double(m) - log(double(s))
                     : (double(x) * double(kLog2e) - double(base_of(m)) - log2(double(s))) / double(kLog2e);
    } else {
      s = __builtin_nanf("");
      sum = __builtin_nan("");
    }
    info[t].top = m;
    info[t].sum = s > 0.0f ? s : __builtin_nanf("");
  }
  __shared__ double wsum[kPfSeqThreads / 64];
  __shared__ int wcount[kPfSeqThreads / 64];
  __shared__ bool last;
  sum = wave_sum(sum);
  count = wave_sum(count);
  if ((threadIdx.x & 63) == 0) {
    wsum[threadIdx.x >> 6] = sum;
    wcount[threadIdx.x >> 6] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPfSeqThreads / 64; ++w) {
      sum += wsum[w];
      count += wcount[w];
    }
    const double n = P.average ? double(count > 0 ? count : 1) : 1.0;
    sum /= n;
    logps[i] = float(sum);
    if (!P.pairs) {
      coef[i] = float(1.0 / n);
    } else {
      __hip_atomic_store(sums + 2 * i, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(sums + 2 * i + 1, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == unsigned(L.S - 1);
    }
  }
  if (!P.pairs) return;
  __syncthreads();
  if (!last) return;
  const int64_t pairs = L.S / 2;
  double total = 0.0;
  for (int64_t p = threadIdx.x; p < pairs; p += kPfSeqThreads) {
    double v[2], n[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t q = p + k * pairs;
      v[k] = __hip_atomic_load(sums + 2 * q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) - (P.ref ? double(P.ref[q]) : 0.0);
      n[k] = __hip_atomic_load(sums + 2 * q + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const double beta = P.beta, eps = P.eps, d = beta * (v[0] - v[1]);
    // a side of weight 0 is not there: 0 times the infinity of an answer that the model cannot give
    // is none (both sides computed: 1 us less than a branch each, which computes their log twice)
    const double near = softplus(-d), far = softplus(d);
    total += (eps < 1.0 ? (1.0 - eps) * near : 0.0) + (eps > 0.0 ? eps * far : 0.0);
    const double up = exp(-near), down = exp(-far);  // sigmoids of d and -d
    const double c = beta / double(pairs) * (eps * up - (1.0 - eps) * down);
    coef[p] = float(c / n[0]);
    coef[p + pairs] = float(-c / n[1]);
  }
  total = wave_sum(total);
  __syncthreads();  // wsum's sequence sums are read
  if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kPfSeqThreads / 64; ++w) total += wsum[w];
    *loss = float(total / double(pairs));
  }
}

// dz = c ([v = y] - softmax), c = coef[seq] * (grad, or grad[seq] per sequence).  LINES: the
// gradient's rows are whole 64-byte lines.
template <int XT, bool LINES>
__global__ __launch_bounds__(kPfThreads) void logits_grad_kernel(Rows r, const void* z, int splits, const RowInfo* info,
                                                                 const float* coef, const float* grad, bool per_seq,
                                                                 void* dz, int64_t lddz) {
  typedef typename Elem<XT>::T T;
  constexpr int VW = Elem<XT>::kVec;
  const int64_t t = blockIdx.x / unsigned(splits);
  const int split = int(blockIdx.x % unsigned(splits));
  const RowInfo I = info[t];
  const T* row = static_cast<const T*>(z) + r.at(t);
  T* out = static_cast<T*>(dz) + t * lddz;
  const Piece<XT> p = piece_of<XT>(r.V, split, splits);
  constexpr int64_t kSpan = int64_t(kPfThreads) * VW;
  int64_t v = p.v0 + threadIdx.x * VW;
  if (I.target == -1) {
    const float zero[VW] = {};
    for (; v < p.v1; v += kSpan) {
      if constexpr (LINES) store16<true>(out + v, u32x4{0u, 0u, 0u, 0u});
      else store16_part<XT>(out + v, zero, p.v1 - v);
    }
    return;
  }
  float c = coef[I.seq];
  if (grad) c *= per_seq ? grad[I.seq] : grad[0];
  const float k = -c / I.sum, base = base_of(I.top);
  const bool equal = huge(I.top);  // of the row
  auto put = [&](float (&f)[VW], int64_t at, int64_t n) {
    float e[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) {
      e[i] = equal ? (f[i] == I.top ? 1.0f : 0.0f) : term(f[i], base);
      f[i] = k * e[i];
    }
    const int64_t y = I.target - at;
    if (y >= 0 && y < VW) {
      // the label's 1 - p cancels: p by a division, 1 where nothing stands beside it
#pragma unroll
      for (int i = 0; i < VW; ++i)
        if (i == y) f[i] = c * (1.0f - e[i] / I.sum);
    }
    if constexpr (LINES) store16<true>(out + at, pack16<XT>(f));
    else store16_part<XT>(out + at, f, n);
  };
  for (; v + (kPfUnroll - 1) * kSpan + VW <= p.v1; v += kPfUnroll * kSpan) {
    u32x4 raw[kPfUnroll];
#pragma unroll
    for (int u = 0; u < kPfUnroll; ++u) raw[u] = load16_any(row + v + u * kSpan);
#pragma unroll
    for (int u = 0; u < kPfUnroll; ++u) {
      float f[VW];
      unpack16<XT>(raw[u], f);
      put(f, v + u * kSpan, VW);
    }
  }
  for (; v < p.v1; v += kSpan) {
    float f[VW];
    unpack16<XT>(load16_part<XT>(row + v, p.v1 - v), f);
    put(f, v, p.v1 - v);
  }
}

// Workgroups of a row: pieces of `piece` bytes; fewer rows than fill the GPU are split until
// there are about four workgroups a compute unit, or pieces of 8 KiB.
int row_splits(int64_t T, int64_t V, int es, int64_t piece) {
  const int64_t want = std::min<int64_t>(ceil_div(4 * int64_t(device_cus()), std::max<int64_t>(T, 1)), 64);
  return int(std::max(ceil_div(V * es, piece), std::min(want, ceil_div(V * es, int64_t(8192)))));
}
// Bytes of a row that a workgroup takes.  Replayed from a graph, 4862 rows of 256 KB forward (both
// launches): 237 us in pieces of 128 KiB, 242 in 64, 254 in 32, 240 whole; their gradient and 3474
// rows of zeros: 648 us in pieces of 32 KiB, 654 in 64, 669 in 128.
constexpr int64_t kSumsPiece = 128 << 10, kGradPiece = 32 << 10;

size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

int check_rows(int dtype, int64_t T, int64_t V, int64_t ld, int64_t period, int64_t outer, Rows* r) {
  if (!valid_float_dtype(dtype)) return RQ_ERR_BAD_DTYPE;
  if (T < 0 || V < 1 || V > INT32_MAX || ld < V || period < 0 || (period > 0 && outer < 0)) return RQ_ERR_BAD_SHAPE;
  if (T > kMaxThreads1D / kPfThreads) return RQ_ERR_UNSUPPORTED;  // workgroups of one launch
  *r = Rows{T, V, ld, period, outer};
  return RQ_OK;
}

}  // namespace
}  // namespace rq

extern "C" int rq_preference_workspace_size(int dtype, int64_t T, int64_t V, int64_t S, int64_t* bytes) {
  using namespace rq;
  if (!bytes) return RQ_ERR_NULL_POINTER;
  if (!valid_float_dtype(dtype)) return RQ_ERR_BAD_DTYPE;
  if (T < 0 || V < 1 || S < 1) return RQ_ERR_BAD_SHAPE;
  *bytes = int64_t(256 + up256(size_t(S) * 16) + up256(size_t(T) * row_splits(T, V, int(dtype_size(dtype)), kSumsPiece) * 8));
  return RQ_OK;
}

extern "C" int rq_preference_forward(const void* logits, int dtype, int64_t T, int64_t V, int64_t ld, int64_t period,
                                     int64_t outer, const int64_t* labels, const int32_t* offsets, int64_t S,
                                     int64_t ignore_index, const float* ref_logps, float beta, float label_smoothing,
                                     int average, float* logps, float* loss, float* coef, void* row_info,
                                     void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace rq;
  Rows r{};
  int st = check_rows(dtype, T, V, ld, period, outer, &r);
  if (st != RQ_OK) return st;
  if (T < 1 || S < 1 || S > kMaxThreads1D / kPfSeqThreads || (loss && S % 2 != 0) || (!offsets && T % S != 0)) return RQ_ERR_BAD_SHAPE;
  if (!logps || !coef || !workspace || !logits || !labels || !row_info) return RQ_ERR_NULL_POINTER;
  const int es = int(dtype_size(dtype)), splits = row_splits(T, V, es, kSumsPiece);
  int64_t need = 0;
  if ((st = rq_preference_workspace_size(dtype, T, V, S, &need)) != RQ_OK) return st;
  if (workspace_bytes < need) return RQ_ERR_WORKSPACE;
  if (!aligned(workspace, 256) || !aligned(row_info, 16) || !aligned(logits, es)) return RQ_ERR_BAD_ALIGNMENT;
  char* ws = static_cast<char*>(workspace);
  uint32_t* done = reinterpret_cast<uint32_t*>(ws);
  double* sums = reinterpret_cast<double*>(ws + 256);
  float* part = reinterpret_cast<float*>(ws + 256 + up256(size_t(S) * 16));
  RowInfo* info = static_cast<RowInfo*>(row_info);
  const Labels L{labels, offsets, S, ignore_index};
  const Pairs P{ref_logps, beta, label_smoothing, average != 0, loss != nullptr};
  if (T * splits > kMaxThreads1D / kPfThreads) return RQ_ERR_UNSUPPORTED;
  const unsigned grid = unsigned(T * splits);
  RQ_DISPATCH_DT(dtype, XT, row_sums_kernel<XT><<<grid, kPfThreads, 0, stream>>>(r, L, logits, splits, info, part, done));
  if ((st = rq_check_launch()) != RQ_OK) return st;
  RQ_DISPATCH_DT(dtype, XT, sequences_kernel<XT><<<unsigned(S), kPfSeqThreads, 0, stream>>>(
                                r, L, logits, splits, info, part, done, sums, P, logps, loss, coef));
  return rq_check_launch();
}

extern "C" int rq_preference_backward(const void* logits, int dtype, int64_t T, int64_t V, int64_t ld, int64_t period,
                                      int64_t outer, const void* row_info, const float* coef, const float* grad,
                                      int grad_per_sequence, void* dlogits, int64_t lddz, hipStream_t stream) {
  using namespace rq;
  Rows r{};
  const int st = check_rows(dtype, T, V, ld, period, outer, &r);
  if (st != RQ_OK) return st;
  if (lddz < V) return RQ_ERR_BAD_SHAPE;
  if (T == 0) return RQ_OK;
  if (!logits || !row_info || !coef || !dlogits) return RQ_ERR_NULL_POINTER;
  const int es = int(dtype_size(dtype));
  if (!aligned(row_info, 16) || !aligned(logits, es) || !aligned(dlogits, es)) return RQ_ERR_BAD_ALIGNMENT;
  const int splits = row_splits(T, V, es, kGradPiece);
  if (T * splits > kMaxThreads1D / kPfThreads) return RQ_ERR_UNSUPPORTED;
  const unsigned grid = unsigned(T * splits);
  const RowInfo* info = static_cast<const RowInfo*>(row_info);
  if (aligned(dlogits, 64) && lddz * es % 64 == 0 && V * es % 64 == 0)
    RQ_DISPATCH_DT(dtype, XT, logits_grad_kernel<XT, true><<<grid, kPfThreads, 0, stream>>>(
                                  r, logits, splits, info, coef, grad, grad_per_sequence != 0, dlogits, lddz));
  else
    RQ_DISPATCH_DT(dtype, XT, logits_grad_kernel<XT, false><<<grid, kPfThreads, 0, stream>>>(
                                  r, logits, splits, info, coef, grad, grad_per_sequence != 0, dlogits, lddz));
  return rq_check_launch();
}
