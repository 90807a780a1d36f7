// Entry points of the linears on MXFP4 weights: argument checks and the choice of kernel.
#include "rq_mx4.h"

namespace rq {

int mx4_compute_units(int* cus);

namespace {

// Whether a forward call runs on the kernel for few rows (us, it and the tiles).  One weight: up to 32 rows where the
// contraction is not long (4096 -> 4096 with 16 rows 8 and 16, with 32 13 and 16; 8192 -> 2048 with 24 rows 18 and 18, with 32
// 21 and 18; 11008 -> 4096 with 16 rows 20 and 21, with 24 24 and 22); fp32 rows up to 16 (4096 -> 14336 with 16 rows 21 and 41,
// with 24 54 and 42); 4-bit activations up to 64 (4096 -> 14336 with 33 rows 20 and 20, with 64 23 and 23; 4096 -> 4096 12
// and 17, 14 and 20).  Experts: up to 8 rows each on average, fp32 rows 16 (16 of 4096 -> 2048 with 128 rows 24 and 44, with 256
// 44 and 36; 64 of 4096 -> 8192 with 512 328 and 347, with 768 387 and 351; fp32 16 of 4096 -> 2048 with 256 rows 68 and 90).
bool few(const MxCall& c) {
  if (c.dx || ceil_div(c.M, c.xdiv) * mx_pad(c.wk) * int64_t(dtype_size(c.dt)) > int64_t(kMxFewBytes)) return false;
  if (c.rows.p) return c.M <= (c.dt == RQ_DTYPE_F32 ? 16 : 8) * c.E;
  return c.a4 ? c.M <= kTileRows : c.M <= (c.dt == RQ_DTYPE_F32 ? 16 : 32) && c.M * mx_pad(c.wk) <= 24 * 8192;
}

// Sizes, whatever the pointers.  shared: rows of the product that one row of the narrower side stands for.
int check_sizes(int dtype, int64_t M, int64_t K, int64_t N, int64_t E, int64_t shared, bool grouped, int act_bits, bool dx) {
  if (!valid_float_dtype(dtype)) return RQ_ERR_BAD_DTYPE;
  if (M < 0 || K < 1 || N < 1 || E < 1 || shared < 1 || M % shared != 0) return RQ_ERR_BAD_SHAPE;
  if (act_bits != 16 && act_bits != 4) return RQ_ERR_UNSUPPORTED;
  if (!grouped && (E != 1 || shared != 1)) return RQ_ERR_BAD_SHAPE;
  if (grouped && act_bits == 4) return RQ_ERR_UNSUPPORTED;
  // 32-bit offsets within 64 rows of a tile (mg_plan: taller tiles; rows of x, of at most 2^24, need no check) and a
  // weight's scales
  if (E > kMaxAdapters || M > (int64_t(1) << 30) || K > (int64_t(1) << 24) || N > (int64_t(1) << 30) ||
      mx_pad(K) * ceil_div(N, 64) > (int64_t(1) << 29) ||
      (dx && !mx_rows_reached(M < kTileRows ? M : kTileRows, ceil_div(N, 64) * 64)))
    return RQ_ERR_UNSUPPORTED;
  return RQ_OK;
}

int64_t scratch_of(const MxCall& c, int cus) {
  if (few(c)) return mx4_few_scratch(c);
  return c.a4 ? mx4_a4_scratch(c, cus) : mx4_gemm_scratch(c, cus);
}

MxCall call_of(int dtype, int64_t M, int64_t K, int64_t N, int64_t E, int64_t shared, const void* plan, int act_bits, bool dx,
               int64_t ldx, bool aligned16) {
  MxCall c{};
  c.dt = dtype;
  c.M = M;
  c.E = E;
  c.N = N;
  c.wk = K;
  c.K = dx ? N : K;
  c.ldx = ldx;
  c.aligned16 = aligned16 && ldx * int64_t(dtype_size(dtype)) % 16 == 0;
  c.xdiv = dx ? 1 : int(shared);
  c.ysum = dx ? int(shared) : 1;
  c.rows = rows_plan(static_cast<const int32_t*>(plan), M, E);
  c.a4 = act_bits == 4;
  c.dx = dx;
  return c;
}

int run(MxCall& c, const void* x, int64_t plan_bytes, const uint8_t* codes, const uint8_t* scales,
        const void* bias, void* y, int64_t ldy, void* scratch, int64_t scratch_bytes, hipStream_t stream) {
  if (c.ldx < c.K || ldy < (c.dx ? c.wk : c.N)) return RQ_ERR_BAD_SHAPE;
  if (c.M == 0) return RQ_OK;
  if (!x || !codes || !scales || !y) return RQ_ERR_NULL_POINTER;
  if (c.rows.p && plan_bytes < 4 * c.rows.words()) return RQ_ERR_WORKSPACE;
  const size_t es = dtype_size(c.dt);
  if (!aligned(x, es) || !aligned(y, es) || !aligned(bias, es) || !aligned(codes, 16) || !aligned(scales, 4) ||
      !aligned(c.rows.p, 16))
    return RQ_ERR_BAD_ALIGNMENT;
  int cus = 0;
  const int st = mx4_compute_units(&cus);
  if (st != RQ_OK) return st;
  const int64_t need = scratch_of(c, cus);
  if (need > 0 && !scratch) return RQ_ERR_NULL_POINTER;
  if (scratch_bytes < need) return RQ_ERR_WORKSPACE;
  if (need > 0 && !aligned(scratch, 256)) return RQ_ERR_BAD_ALIGNMENT;
  c.x = x;
  c.codes = codes;
  c.scales = scales;
  c.bias = bias;
  c.y = y;
  c.ldy = ldy;
  c.scratch = scratch;
  c.stream = stream;
  if (few(c)) return mx4_few_run(c);
  return c.a4 ? mx4_a4_run(c, cus) : mx4_gemm_run(c, cus);
}

}  // namespace

// Of the current device, asked for once.
int mx4_compute_units(int* cus) {
  static std::atomic<int> known[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return RQ_ERR_HIP;
  if (dev < 64) {
    *cus = known[dev].load(std::memory_order_relaxed);
    if (*cus > 0) return RQ_OK;
  }
  if (hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return RQ_ERR_HIP;
  if (dev < 64) known[dev].store(*cus, std::memory_order_relaxed);
  return RQ_OK;
}

}  // namespace rq

extern "C" int rq_mx4_linear_scratch_size(int dtype, int64_t M, int64_t K, int64_t N, int64_t E, int64_t shared, int grouped,
                                          int act_bits, int dx, int64_t ldx, int aligned16, int64_t* bytes) {
  using namespace rq;
  if (!bytes) return RQ_ERR_NULL_POINTER;
  int cus = 0;
  int st = check_sizes(dtype, M, K, N, E, shared, grouped != 0, act_bits, dx != 0);
  if (st != RQ_OK) return st;
  if (ldx < (dx ? N : K)) return RQ_ERR_BAD_SHAPE;
  *bytes = 0;
  if (M == 0) return RQ_OK;
  st = mx4_compute_units(&cus);
  if (st != RQ_OK) return st;
  static const int32_t some = 0;  // any non-null plan: sizes alone are asked for
  *bytes = scratch_of(call_of(dtype, M, K, N, E, shared, grouped ? &some : nullptr, act_bits, dx != 0, ldx, aligned16 != 0), cus);
  return RQ_OK;
}

extern "C" int rq_mx4_tile_plan(int dtype, int64_t M, int64_t K, int64_t N, int64_t E, int64_t shared, int grouped, int act_bits,
                                int dx, int64_t ldx, int aligned16, int32_t* out) {
  using namespace rq;
  if (!out) return RQ_ERR_NULL_POINTER;
  const int st = check_sizes(dtype, M, K, N, E, shared, grouped != 0, act_bits, dx != 0);
  if (st != RQ_OK) return st;
  if (M < 1 || ldx < (dx ? N : K)) return RQ_ERR_BAD_SHAPE;
  int cus = 0;
  if (mx4_compute_units(&cus) != RQ_OK) cus = 256;
  static const int32_t some = 0;  // any non-null plan: sizes alone are asked for
  const MxCall c = call_of(dtype, M, K, N, E, shared, grouped ? &some : nullptr, act_bits, dx != 0, ldx, aligned16 != 0);
  out[0] = out[1] = out[2] = 0;
  if (few(c)) return RQ_OK;
  c.a4 ? mx4_a4_tiles(c, cus, out) : mx4_gemm_tiles(c, cus, out);
  return RQ_OK;
}

extern "C" int rq_mx4_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, int64_t shared, const void* plan,
                             int64_t plan_bytes, const uint8_t* codes, const uint8_t* scales, int64_t E, int64_t N,
                             const void* bias, int act_bits, void* y, int64_t ldy, void* scratch, int64_t scratch_bytes,
                             hipStream_t stream) {
  using namespace rq;
  const int st = check_sizes(dtype, M, K, N, E, shared, plan != nullptr, act_bits, false);
  if (st != RQ_OK) return st;
  MxCall c = call_of(dtype, M, K, N, E, shared, plan, act_bits, false, ldx, aligned(x, 16));
  return run(c, x, plan_bytes, codes, scales, bias, y, ldy, scratch, scratch_bytes, stream);
}

extern "C" int rq_mx4_linear_dx(const void* dy, int dtype, int64_t M, int64_t N, int64_t lddy, const void* plan,
                                int64_t plan_bytes, const uint8_t* codes, const uint8_t* scales, int64_t E, int64_t K,
                                int64_t shared, void* dx, int64_t lddx, void* scratch, int64_t scratch_bytes,
                                hipStream_t stream) {
  using namespace rq;
  const int st = check_sizes(dtype, M, K, N, E, shared, plan != nullptr, 16, true);
  if (st != RQ_OK) return st;
  MxCall c = call_of(dtype, M, K, N, E, shared, plan, 16, true, lddy, aligned(dy, 16));
  return run(c, dy, plan_bytes, codes, scales, nullptr, dx, lddx, scratch, scratch_bytes, stream);
}
