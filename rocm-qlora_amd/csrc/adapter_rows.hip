// Grouping a batch's rows by adapter (rq_rows.h): a counting sort in one
// workgroup, stable and without an atomic whose order shows.  Each of eight waves
// counts its own stretch of the rows, the counts are summed over waves and
// adapters, and each wave then places its stretch 64 rows at a time, rows of the
// same adapter found by a ballot for each bit of its number.  Bound by latency, the chain of
// loads, counts and sums: 3.6 us for 8 rows, 4.9 for 256 rows of 64 adapters, 7.4 for 4096 of
// 4, 35 for 4096 of 1024 (one of two tables after the other, sums by lane shuffles, padding a
// tile a thread: 6.6, 7.5, 10 and 63; a graph's replays).
// It runs once for a batch, for all the projections of all its layers.
#include "rq_launch.h"
#include "rq_rows.h"

namespace rq {
namespace {

constexpr int kArThreads = 512;
constexpr int kArWaves = kArThreads / 64;

__device__ __forceinline__ int adapter_of(const int32_t* ids, int64_t row, int n) {
  const int a = ids[row];
  return a >= 0 && a < n ? a : n;  // n: no adapter
}

// Exclusive sums of v over 64 lanes, carry in and out: shifts by 1, 2, 4 and 8 within the rows
// of 16 lanes, then the sums of the rows before.
__device__ __forceinline__ int wave_excl(int v, int& carry) {
  int s = v;
  s += __builtin_amdgcn_update_dpp(0, s, 0x111, 0xF, 0xF, true);
  s += __builtin_amdgcn_update_dpp(0, s, 0x112, 0xF, 0xF, true);
  s += __builtin_amdgcn_update_dpp(0, s, 0x114, 0xF, 0xF, true);
  s += __builtin_amdgcn_update_dpp(0, s, 0x118, 0xF, 0xF, true);
  s += __builtin_amdgcn_update_dpp(0, s, 0x142, 0xA, 0xF, false);  // lane 15 to the next row, 47 to the last
  s += __builtin_amdgcn_update_dpp(0, s, 0x143, 0xC, 0xF, false);  // lane 31 to the upper half
  const int e = carry + s - v;
  carry += __builtin_amdgcn_readlane(s, 63);
  return e;
}

__global__ __launch_bounds__(kArThreads) void adapter_rows_kernel(const int32_t* ids, RowsPlan P, int32_t* plan) {
  __shared__ int hist[kArWaves][kMaxAdapters + 1];  // counts, then this wave's next place among the adapter's rows
  __shared__ int first[kMaxAdapters + 2];           // first tile of each adapter
  __shared__ int total[kMaxAdapters + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = P.n;
  const int64_t M = P.M;
  const int64_t per = ceil_div(ceil_div(M, kArWaves), 64) * 64;
  const int64_t r0 = per * wave < M ? per * wave : M, r1 = r0 + per < M ? r0 + per : M;
  const int id0 = r0 + lane < r1 ? adapter_of(ids, r0 + lane, n) : 0;  // of the stretch's first 64 rows
  for (int w = 0; w < kArWaves; ++w)
    for (int a = tid; a <= n; a += kArThreads) hist[w][a] = 0;
  __syncthreads();
  if (r0 + lane < r1) atomicAdd(&hist[wave][id0], 1);
  int64_t q = r0 + lane + 64;
  for (; q + 192 < r1; q += 256) {  // four loads in flight
    int a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = adapter_of(ids, q + 64 * i, n);
#pragma unroll
    for (int i = 0; i < 4; ++i) atomicAdd(&hist[wave][a[i]], 1);
  }
  for (; q < r1; q += 64) atomicAdd(&hist[wave][adapter_of(ids, q, n)], 1);
  __syncthreads();
  for (int a = tid; a <= n; a += kArThreads) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < kArWaves; ++w) {
      const int c = hist[w][a];
      hist[w][a] = s;
      s += c;
    }
    total[a] = s;
  }
  __syncthreads();
  if (wave == 0) {
    int carry = 0;
    for (int a0 = 0; a0 <= n; a0 += 64) {
      const int a = a0 + lane;
      const int e = wave_excl(a <= n ? (total[a] + kTileRows - 1) / kTileRows : 0, carry);
      if (a <= n) first[a] = e;
    }
    if (lane == 0) first[n + 1] = carry;
  }
  __syncthreads();
  const int tiles = first[n + 1];
  // chunks of the adapters' tiles (an empty one for an adapter without rows, none for the rows
  // without one), and the partial slots of adapters with several: a table by each of the last
  // waves, which have the fewest rows
  const int k = kArWaves - 1 - wave;
  if (k < kChunkTables) {
    int chunks = 0, parts = 0;
    int32_t* tab = plan + P.off_chunks() + 4 * int64_t(P.C) * k;
    int32_t* part = plan + P.off_part() + 2 * int64_t(n) * k;
    for (int a0 = 0; a0 < n; a0 += 64) {
      const int a = a0 + lane;
      const int mine = a < n ? (total[a] + kTileRows - 1) / kTileRows : 0;
      const Chunks ch = adapter_chunks(mine, tiles, k);
      const int c = a < n ? ch.n : 0;
      const int c0 = wave_excl(c, chunks), p0 = wave_excl(c > 1 ? c : 0, parts);
      const int t0 = a < n ? first[a] : 0;
      if (a < n) {
        part[2 * a] = c;
        part[2 * a + 1] = p0;
      }
      for (int i = 0; i < c; ++i) {
        const int b = t0 + i * ch.tiles, e = b + ch.tiles < t0 + mine ? b + ch.tiles : t0 + mine;
        tab[4 * (c0 + i)] = a;
        tab[4 * (c0 + i) + 1] = b;
        tab[4 * (c0 + i) + 2] = e;
        tab[4 * (c0 + i) + 3] = c > 1 ? p0 + i : -1;
      }
    }
    if (lane == 0) plan[1 + k] = chunks;
  }
  if (tid < 16 && (tid == 0 || tid > kChunkTables)) plan[tid] = tid == 0 ? tiles : 0;
  for (int t = tid; t < tiles; t += kArThreads) {
    int lo = 0, hi = n;  // the last adapter whose first tile is at most t
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (first[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    const int left = total[lo] - kTileRows * (t - first[lo]);
    plan[16 + 2 * t] = lo < n ? lo : -1;
    plan[16 + 2 * t + 1] = left < kTileRows ? left : kTileRows;
  }
  for (int a = wave; a <= n; a += kArWaves) {  // the slots after the last row of an adapter
    const int left = total[a] % kTileRows;
    if (left > 0 && lane >= left) plan[P.off_rows() + int64_t(kTileRows) * (first[a] + total[a] / kTileRows) + lane] = -1;
  }
  for (int t = tiles + tid; t < P.T; t += kArThreads) {
    plan[16 + 2 * t] = -1;
    plan[16 + 2 * t + 1] = 0;
  }
  const int bits = 32 - __clz(n);
  int next = id0;
  for (int64_t b = r0; b < r1; b += 64) {
    const int64_t r = b + lane;
    const bool on = r < r1;
    const int a = next;
    next = r + 64 < r1 ? adapter_of(ids, r + 64, n) : 0;
    unsigned long long same = __ballot(on);  // the lanes with this one's adapter: alike in every bit
    for (int k = 0; k < bits; ++k) {
      const unsigned long long set = __ballot(a >> k & 1);
      same &= a >> k & 1 ? set : ~set;
    }
    const unsigned long long before = same & ((1ull << lane) - 1);
    if (on) {
      const int base = hist[wave][a];
      plan[P.off_rows() + int64_t(kTileRows) * first[a] + base + __popcll(before)] = int32_t(r);
      __builtin_amdgcn_wave_barrier();  // all lanes have read before the first of each adapter writes
      if (!before) hist[wave][a] = base + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace
}  // namespace rq

extern "C" int rq_adapter_rows_size(int64_t M, int64_t n, int64_t* bytes) {
  using namespace rq;
  if (!bytes) return RQ_ERR_NULL_POINTER;
  if (M < 0 || n < 1 || M > (int64_t(1) << 30)) return RQ_ERR_BAD_SHAPE;
  if (n > kMaxAdapters) return RQ_ERR_UNSUPPORTED;
  static const int32_t some = 0;  // any non-null plan: sizes alone are asked for
  *bytes = 4 * rows_plan(&some, M, n).words();
  return RQ_OK;
}

extern "C" int rq_adapter_rows(const int32_t* ids, int64_t M, int64_t n, void* plan, int64_t plan_bytes,
                               hipStream_t stream) {
  using namespace rq;
  int64_t need = 0;
  const int st = rq_adapter_rows_size(M, n, &need);
  if (st != RQ_OK) return st;
  if (!plan || (M > 0 && !ids)) return RQ_ERR_NULL_POINTER;
  if (plan_bytes < need) return RQ_ERR_WORKSPACE;
  if (!aligned(plan, 16) || !aligned(ids, 4)) return RQ_ERR_BAD_ALIGNMENT;
  int32_t* p = static_cast<int32_t*>(plan);
  adapter_rows_kernel<<<1, kArThreads, 0, stream>>>(ids, rows_plan(p, M, n), p);
  return rq_check_launch();
}
