// Row accesses of 16 bytes at any element alignment (global loads and stores of
// gfx950 take any byte address; a row of odd length or a strided view needs no
// copy), and the pieces of a row's end.
#pragma once

#include "rq_common.h"
#include "rq_mfma.h"

namespace rq {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

template <int XT>
struct Elem {
  typedef uint16_t T;
  static constexpr int kVec = 8;    // elements of 16 bytes
  static constexpr int kStep = 32;  // contraction of one mma() call
};
template <>
struct Elem<RQ_DTYPE_F32> {
  typedef float T;
  static constexpr int kVec = 4;
  static constexpr int kStep = 16;
};

template <int XT>
__device__ __forceinline__ float to_f32(typename Elem<XT>::T v) {
  if constexpr (XT == RQ_DTYPE_F32) return v;
  else return from_x16<XT>(v);
}
template <int XT>
__device__ __forceinline__ typename Elem<XT>::T from_f32(float v) {
  if constexpr (XT == RQ_DTYPE_F32) return v;
  else return uint16_t(to_x16<XT>(v));
}

__device__ __forceinline__ u32x4 load16_any(const void* p) {
  const u32x4_any v = *static_cast<const u32x4_any*>(p);
  return u32x4{v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ void store16_any(void* p, u32x4 v) {
  *static_cast<u32x4_any*>(p) = u32x4_any{v.x, v.y, v.z, v.w};
}

// Past the caches, for results that no one here reads again: where the lanes of a store fill
// 64-byte lines of memory it leaves the caches to what is read (a fifth faster at times),
// where they do not each line is written in parts (half as fast).
template <bool PAST>
__device__ __forceinline__ void store16(void* p, u32x4 v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, static_cast<u32x4*>(p));
  else store16_any(p, v);
}

// Less than 16 bytes, element by element: the ends of rows.  Not inlined: the addresses of
// the elements would take registers from the loops around.
template <int XT>
__attribute__((noinline)) __device__ u32x4 load_edge(const typename Elem<XT>::T* p, int n) {
  u32x4 v = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < Elem<XT>::kVec; ++i) {
    if (i >= n) break;
    if constexpr (XT == RQ_DTYPE_F32) v[i] = f2u(p[i]);
    else v[i >> 1] |= uint32_t(p[i]) << (16 * (i & 1));
  }
  return v;
}
template <int XT>
__attribute__((noinline)) __device__ void store_edge(typename Elem<XT>::T* p, u32x4 v, int n) {
#pragma unroll
  for (int i = 0; i < Elem<XT>::kVec; ++i) {
    if (i >= n) break;
    if constexpr (XT == RQ_DTYPE_F32) p[i] = u2f(v[i]);
    else p[i] = uint16_t(v[i >> 1] >> (16 * (i & 1)));
  }
}

// The first `n` elements at p (n <= 0: none) as 16 bytes, zeros after them.
template <int XT>
__device__ __forceinline__ u32x4 load16_part(const typename Elem<XT>::T* p, int64_t n) {
  if (n >= Elem<XT>::kVec) return load16_any(p);
  return load_edge<XT>(p, int(n));
}

// 16 bytes as fp32 values, and back (rounded to nearest even).
template <int XT>
__device__ __forceinline__ void unpack16(const u32x4& v, float (&f)[Elem<XT>::kVec]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (XT == RQ_DTYPE_F32) {
      f[i] = u2f(v[i]);
    } else {
      f[2 * i] = from_x16<XT>(v[i] & 0xFFFFu);
      f[2 * i + 1] = from_x16<XT>(v[i] >> 16);
    }
  }
}
template <int XT>
__device__ __forceinline__ u32x4 pack16(const float (&f)[Elem<XT>::kVec]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (XT == RQ_DTYPE_F32) v[i] = f2u(f[i]);
    else v[i] = cvt_pk<XT>(f[2 * i], f[2 * i + 1]);
  }
  return v;
}

template <int XT>
__device__ __forceinline__ void store16_part(typename Elem<XT>::T* p, const float (&f)[Elem<XT>::kVec], int64_t n) {
  if (n >= Elem<XT>::kVec) store16_any(p, pack16<XT>(f));
  else store_edge<XT>(p, pack16<XT>(f), int(n));
}

// acc += A B over kStep contraction steps, both operands as 16 bytes a lane: lane
// (i, g) = (l % 16, l / 16) holds A[i][V g + e] and B[V g + e][i], e < V = kVec;
// register r of the result is D[4 g + r][i].
template <int XT>
__device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, f32x4 acc) {
  if constexpr (XT == RQ_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(a[e]), u2f(b[e]), acc, 0, 0, 0);
    return acc;
  } else {
    return mfma16x16x32<XT>(a, b, acc);
  }
}

}  // namespace rq
