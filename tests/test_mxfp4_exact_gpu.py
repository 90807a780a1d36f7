"""MXFP4 linears on operands whose products and sums are exact: small whole numbers beside every code at scales of 1/2, 1
and 2, so that a sum in any order is the same, as long as it stays under 2^22.  Results are equal, whatever the length."""
import ctypes
import functools

import pytest
import torch

import mxfp4_oracle as oracle
from rocm_qlora import ExpertRows, MXFP4Tensor, dequantize_mxfp4, mxfp4_expert_linear, mxfp4_linear, ops
from rocm_qlora import _native as nat

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def exact_weight(N, K, dev, seed=0, scales=(126, 129)):
    """A weight [N, K] of every code, and its values in fp64 (made on the GPU: it may be large)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    pitch = ops.mx4_pad(K)
    codes = torch.randint(0, 256, (N, pitch // 2), dtype=torch.uint8, device=dev, generator=g)
    codes[:, (K + 1) // 2:] = 0
    if K % 2:
        codes[:, K // 2] &= 15
    return MXFP4Tensor(codes, torch.randint(*scales, (N, pitch // 32), dtype=torch.uint8, device=dev, generator=g), K)


def whole(M, K, dtype, dev, seed=1, most=2):
    """Rows of whole numbers of at most `most` in magnitude."""
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randint(-most, most + 1, (M, K), dtype=torch.int8, device=dev, generator=g).to(dtype)


def test_rows_past_4_gib_in_a_copied_tile(dev):
    """512 rows of 18 MB: the rows are copied, and the copy's tiles hold no more of them than 32-bit offsets reach."""
    M, K, N = 512, 9_000_064, 2048
    print("rows of 18 MB", M, K, N, flush=True)
    w = exact_weight(N, K, dev, 1, (127, 128))
    x = whole(M, K, BF16, dev, 2, 1)
    y = mxfp4_linear(x, w)
    want = torch.zeros(M, 16, dtype=torch.float64, device=dev)
    cols = torch.arange(0, N, N // 16, device=dev)
    step = 1 << 17
    for k in range(0, K, step):
        e = min(K, k + step)
        part = MXFP4Tensor(w.codes[cols, k // 2:-(-e // 128) * 64].contiguous(), w.scales[cols, k // 32:-(-e // 128) * 4].contiguous(), e - k)
        want += (x[:, k:e].float() @ dequantize_mxfp4(part, FP32).t()).double()
    assert float(want.abs().max()) < 2.0 ** 20
    assert torch.equal(y[:, cols], want.to(BF16))
    # the same rows 64 at a time
    for m in range(0, M, 64):
        assert torch.equal(y[m:m + 64], mxfp4_linear(x[m:m + 64], w)), m


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K,N", [(64, 1408, 4096), (64, 128, 100), (64, 1152, 8192), (64, 640, 14336), (32, 1408, 512), (16, 384, 512)])
def test_scratch_of_its_size_alone(dev, M, K, N, dtype):
    """4-bit activations, an odd number of 128-value steps: their codes and scales fill the scratch memory to its last
    byte where M is 64, and nothing behind it is asked for (it holds what would be NaN scales)."""
    w = exact_weight(N, K, dev, 3)
    x = whole(M, K, dtype, dev, 4)
    xq = torch.from_numpy(oracle.quantize(x)[2])[:, :K]
    want = xq.double() @ oracle.held(w.codes, w.scales, K).t()
    code = nat.dtype_code(dtype)
    n = ctypes.c_int64(0)
    nat.call("rq_mx4_linear_scratch_size", code, M, K, N, 1, 1, 0, 4, 0, K, 1, ctypes.byref(n))
    area = torch.full((n.value + 512,), 255, dtype=torch.uint8, device=dev)
    assert area.data_ptr() % 256 == 0
    y = torch.empty(M, N, dtype=dtype, device=dev)
    nat.call("rq_mx4_linear", x.data_ptr(), code, M, K, K, 1, None, 0, w.codes.data_ptr(), w.scales.data_ptr(), 1, N, None, 4,
             y.data_ptr(), N, area.data_ptr(), n.value, nat.stream_handle(dev))
    assert torch.equal(y.cpu(), want.to(dtype))
    assert bool((area[n.value:] == 255).all())


# ---- long contractions -----------------------------------------------------------------
# splits of the contraction, refills of the scales, the ring's places and the last steps are all passed many times; a
# result that leaves out or repeats one block differs
LONG = [(1 << 18, 33), (200_037, 40), (64, 1 << 17), (130, 100_001), (70_016, 257)]


@functools.lru_cache(maxsize=1)
def long_weight(N, K, dev):
    w = exact_weight(N, K, dev, 5)
    return w, oracle.held(w.codes, w.scales, K)


@pytest.mark.parametrize("M", [2, 20, 100, 300])
@pytest.mark.parametrize("K,N", LONG)
def test_long_contractions(dev, K, N, M):
    w, vals = long_weight(N, K, dev)
    x, dy = whole(M, K, FP32, dev, 6), whole(M, N, FP32, dev, 7)
    want, dwant = x.double().cpu() @ vals.t(), dy.double().cpu() @ vals
    for t in (want, dwant):  # (fp16 holds them, and one block's part is not lost in a result's rounding)
        assert 8.0 < float(t.std()) and float(t.abs().max()) < 2.0 ** 15
    for dtype in (BF16, FP16, FP32):
        assert torch.equal(mxfp4_linear(x.to(dtype), w).cpu(), want.to(dtype)), dtype
        # (whole numbers of at most 2 are MXFP4 values)
        assert torch.equal(mxfp4_linear(x.to(dtype), w, activation_bits=4).cpu(), want.to(dtype)), dtype
        assert torch.equal(ops.mx4_linear_dx(dy.to(dtype), w.codes, w.scales, K).cpu(), dwant.to(dtype)), dtype


@pytest.mark.parametrize("T,k,n", [(3, 2, 2), (70, 2, 3), (300, 1, 2)])
@pytest.mark.parametrize("K,N", [(70_016, 40), (96, 50_001)])
def test_long_contractions_of_experts(dev, K, N, T, k, n):
    w = exact_weight(n * N, K, dev, 8)
    vals = oracle.held(w.codes, w.scales, K).view(n, N, K)
    w = MXFP4Tensor(w.codes.view(n, N, -1), w.scales.view(n, N, -1), K)
    ids = torch.randint(-1, n, (T, k), generator=torch.Generator().manual_seed(T))
    x, dy = whole(T, K, FP32, dev, 9), whole(T * k, N, FP32, dev, 10)
    want, dwant = torch.zeros(T * k, N, dtype=torch.float64), torch.zeros(T * k, K, dtype=torch.float64)
    x64, dy64, flat = x.double().cpu().repeat_interleave(k, 0), dy.double().cpu(), ids.view(-1)
    for e in range(n):
        want[flat == e] = x64[flat == e] @ vals[e].t()
        dwant[flat == e] = dy64[flat == e] @ vals[e]
    dwant = dwant.view(T, k, K).sum(1)
    assert float(want.std()) > 8.0 and float(dwant.std()) > 8.0
    rows = ExpertRows(ids.to(dev), n)
    for dtype in (BF16, FP16, FP32):
        xg = x.to(dtype).requires_grad_(True)
        y = mxfp4_expert_linear(xg, w, rows)
        assert torch.equal(y.detach().cpu(), want.to(dtype)), dtype
        (dx,) = torch.autograd.grad(y, xg, dy.to(dtype))
        assert torch.equal(dx.cpu(), dwant.to(dtype)), dtype


# ---- gradients against differences ------------------------------------------------------
@pytest.mark.parametrize("K,N,T", [(192, 80, 70), (1000, 301, 33), (128, 640, 5), (320, 96, 300)])
@pytest.mark.parametrize("kind", ["linear", "experts"])
def test_gradient_equals_differences(dev, kind, K, N, T):
    """The map is linear: c . (f(x + h v) - f(x - h v)) = 2 h dx . v for every token, on operands that keep both sides exact
    (fp32 sums of multiples of 1/32 that stay under 2^19): equal, not near."""
    k, n, h = (1, 1, 0.25) if kind == "linear" else (2, 3, 0.25)
    w = exact_weight(n * N, K, dev, 11)
    if kind == "linear":
        f = lambda z: mxfp4_linear(z, w)  # noqa: E731
    else:
        w = MXFP4Tensor(w.codes.view(n, N, -1), w.scales.view(n, N, -1), K)
        rows = ExpertRows(torch.randint(0, n, (T, k), generator=torch.Generator().manual_seed(T)).to(dev), n)
        f = lambda z: mxfp4_expert_linear(z, w, rows)  # noqa: E731
    x, v, c = whole(T, K, FP32, dev, 12), whole(T, K, FP32, dev, 13), whole(T * k, N, FP32, dev, 14)
    xg = x.clone().requires_grad_(True)
    y = f(xg)
    (dx,) = torch.autograd.grad(y, xg, c)
    with torch.no_grad():
        diff = ((f(x + h * v) - f(x - h * v)).double() * c.double()).view(T, k * N).sum(1) / (2 * h)
    want = (dx.double() * v.double()).sum(1)
    assert torch.equal(diff, want)
    assert float(want.abs().median()) > 100.0 and float(y.detach().abs().max()) < 2.0 ** 19


# ---- every tile, on whole numbers -------------------------------------------------------
@pytest.mark.parametrize("M,K,N", [(33, 100, 70), (128, 2048, 1000), (200, 4096, 520), (600, 1024, 1030), (1111, 320, 2333), (2300, 1100, 7700),
                                   (4096, 640, 4100), (3900, 512, 4200)])
def test_tiles(dev, M, K, N):
    w = exact_weight(N, K, dev, 15)
    vals = oracle.held(w.codes, w.scales, K)
    x, dy = whole(M, K, FP32, dev, 16), whole(M, N, FP32, dev, 17)
    want, dwant = x.double().cpu() @ vals.t(), dy.double().cpu() @ vals
    for dtype in (BF16, FP16, FP32):
        for bits in (16, 4):
            assert torch.equal(mxfp4_linear(x.to(dtype), w, activation_bits=bits).cpu(), want.to(dtype)), (dtype, bits)
        assert torch.equal(ops.mx4_linear_dx(dy.to(dtype), w.codes, w.scales, K).cpu(), dwant.to(dtype)), dtype


@pytest.mark.parametrize("T,k,n,K,N,skew", [(9, 2, 64, 256, 100, 0), (40, 8, 64, 640, 200, 0), (700, 2, 8, 512, 1100, 0), (2048, 2, 5, 256, 4200, 3),
                                            (64, 2, 16, 1024, 520, 60), (1000, 1, 3, 300, 700, 2)])
def test_experts_tiles(dev, T, k, n, K, N, skew):
    """Rows spread over the experts, and all but a few of them on one."""
    w = exact_weight(n * N, K, dev, 18)
    vals = oracle.held(w.codes, w.scales, K).view(n, N, K)
    w = MXFP4Tensor(w.codes.view(n, N, -1), w.scales.view(n, N, -1), K)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-1, n, (T, k), generator=g)
    if skew:
        ids = torch.where(torch.randint(0, skew, (T, k), generator=g) > 0, n - 1, ids)
    x, dy, flat = whole(T, K, FP32, dev, 19), whole(T * k, N, FP32, dev, 20), ids.view(-1)
    x64, dy64 = x.double().cpu().repeat_interleave(k, 0), dy.double().cpu()
    want, dwant = torch.zeros(T * k, N, dtype=torch.float64), torch.zeros(T * k, K, dtype=torch.float64)
    for e in range(n):
        want[flat == e] = x64[flat == e] @ vals[e].t()
        dwant[flat == e] = dy64[flat == e] @ vals[e]
    dwant = dwant.view(T, k, K).sum(1)
    rows = ExpertRows(ids.to(dev), n)
    for dtype in (BF16, FP16, FP32):
        assert torch.equal(mxfp4_expert_linear(x.to(dtype), w, rows).cpu(), want.to(dtype)), dtype
        dx = ops.mx4_linear_dx(dy.to(dtype), w.codes, w.scales, K, plan=rows.plan, shared=k)
        assert torch.equal(dx.cpu(), dwant.to(dtype)), dtype
