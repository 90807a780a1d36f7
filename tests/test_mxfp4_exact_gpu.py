"""MXFP4 linears on operands whose products and sums are exact: small whole numbers beside every code at scales of 1/2, 1
and 2, so that a sum in any order is the same, as long as it stays under 2^22.  Results are equal, whatever the length."""
import ctypes

import pytest
import torch

import mxfp4_oracle as oracle
from rocm_qlora import MXFP4Tensor, dequantize_mxfp4, mxfp4_linear, ops
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
    """512 rows of 16 MiB: the rows are copied, and the copy's tiles hold no more of them than 32-bit offsets reach."""
    M, K, N = 512, (1 << 23) + 128, 2048
    print("rows of 16 MiB", M, K, N, flush=True)
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
