"""8-bit activation checkpoints against the format's definition in fp64 on the CPU.
Codes, exponents and values are exact: no tolerance."""
import math

from contextlib import nullcontext

import numpy as np
import pytest
import torch

from rocm_qlora import LoRALinear, QuantLinear, ops
from rocm_qlora.checkpoint import Act8, compress, decompress, saved_in_8_bits

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def oracle(x):
    """codes, exponent bytes, values by the definition, block by block."""
    v = x.detach().double().cpu().numpy()
    M, K = v.shape
    nb = -(-K // 32)
    codes, exps = np.zeros((M, nb * 32), np.int64), np.zeros((M, nb), np.int64)
    out = np.zeros((M, nb * 32))
    pad = np.zeros((M, nb * 32))
    pad[:, :K] = v
    for b in range(nb):
        blk = pad[:, 32 * b:32 * b + 32]
        top = np.abs(blk).max(1)
        for m in range(M):
            if not math.isfinite(top[m]):
                exps[m, b] = 255
                out[m, 32 * b:32 * b + 32] = np.nan
                continue
            e = max(math.frexp(top[m])[1] - 1, -127) if top[m] > 0 else -127
            exps[m, b] = e + 127
            q = np.clip(np.rint(blk[m] * 2.0 ** (6 - e)), -127, 127)
            codes[m, 32 * b:32 * b + 32] = q
            out[m, 32 * b:32 * b + 32] = q * 2.0 ** (e - 6)
    return codes, exps, out[:, :K]


def check(x):
    codes, exps = ops.act8_quantize(x)
    wc, we, wv = oracle(x.reshape(-1, x.shape[-1]))
    assert np.array_equal(codes.cpu().view(torch.int8).long().numpy(), wc)
    assert np.array_equal(exps.cpu().long().numpy(), we)
    got = ops.act8_dequantize(codes, exps, x.shape[-1], x.dtype)
    # exact: the value in fp64 is the value in x's dtype
    assert np.array_equal(got.double().cpu().numpy(), wv, equal_nan=True)
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 48), (4, 100), (33, 1001), (7, 4096), (300, 64)])
def test_codes_and_values(dev, M, K, dtype):
    g = torch.Generator().manual_seed(M * K)
    x = torch.randn(M, K, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g))
    check(x.to(dtype).to(dev))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_values_where_rounding_decides(dev, dtype):
    """Ties, values that round up to 128 steps, powers of two, zeros, subnormals, the largest
    numbers, and blocks with an infinity or a NaN."""
    fi = torch.finfo(dtype)
    rows = [
        [1.0] + [(k + 0.5) / 64 for k in range(31)],       # ties, to even
        [-1.0] + [-(k + 0.5) / 64 for k in range(31)],
        [1.9921875] * 16 + [1.984375] * 8 + [-1.9921875] * 8,  # 127.5 steps and the largest code
        [2.0 ** (k % 12 - 6) for k in range(32)],
        [0.0] * 32,
        [-0.0] * 32,
        [fi.tiny] * 31 + [fi.tiny / 2],
        [fi.smallest_normal / 4, fi.smallest_normal / 8] * 16,
        [fi.max, -fi.max] + [fi.max / 3] * 30,
        [float("inf")] + [1.0] * 31,
        [float("nan")] + [0.0] * 31,
        [0.0] * 31 + [float("-inf")],
    ]
    check(torch.tensor(rows, dtype=torch.float64).to(dtype).to(dev))


def test_strided_and_unaligned_rows(dev):
    wide = torch.randn(9, 80, generator=torch.Generator().manual_seed(0)).to(BF16).to(dev)
    check(wide[:, 3:70])
    check(wide[::2, :64])
    check(wide.t())
    x3 = wide[:, :64].reshape(3, 3, 64)
    c = compress(x3)
    assert c.shape == x3.shape and decompress(c).shape == x3.shape and c.nbytes() == 9 * 66
    assert decompress(compress(wide[:0])).shape == (0, 80)
    assert ops.act8_quantize(wide[4])[0].shape == (1, 96)


def test_more_than_2_to_the_31_values(dev):
    """Offsets past 32 bits: the last rows of a long checkpoint."""
    M, K = 70000, 32768
    x = torch.zeros(M, K, dtype=BF16, device=dev)
    x[-3:] = torch.randn(3, K, generator=torch.Generator().manual_seed(0)).to(BF16).to(dev)
    c = compress(x)
    assert torch.equal(decompress(Act8(c.codes[-3:], c.exponents[-3:], x[-3:].shape, BF16)), check(x[-3:]))
    del x
    assert torch.equal(decompress(c)[-3:], check(decompress(c)[-3:]))


def linear_grads(x, w, dy, context):
    with context:
        y = torch.nn.functional.linear(x * 1.0, w)
    return (y, *torch.autograd.grad(y, (x, w), dy))


@pytest.mark.parametrize("cast", [False, True])
def test_saved_in_8_bits(dev, cast):
    """Inside the block a linear's weight gradient is the one at the held input; what the
    forward returns and the input gradient (the weight, also a cast of it) do not change."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(64, 96, generator=g).to(dev).requires_grad_(True)
    p = torch.nn.Parameter(torch.randn(80, 96, generator=g).to(FP16 if cast else FP32).to(dev))
    w = p.float() if cast else p
    dy = torch.randn(64, 80, generator=g).to(dev)
    y0, dx0, dw0 = linear_grads(x, w, dy, nullcontext())
    y8, dx8, dw8 = linear_grads(x, w, dy, saved_in_8_bits(min_elements=1))
    held = decompress(compress(x)).detach().double()
    assert torch.equal(y0, y8) and torch.equal(dx0, dx8)
    bound = (64 + 8) * 2.0 ** -24 * (dy.double().abs().T @ held.abs())
    assert bool(((dw8.double() - dy.double().T @ held).abs() <= bound).all()) and not torch.equal(dw0, dw8)
    assert torch.equal(linear_grads(x, w, dy, saved_in_8_bits())[2], dw0)  # too small to hold
    # a frozen weight is no activation either
    y = torch.nn.functional.linear(x * 1.0, w.detach().half().float())
    with saved_in_8_bits(min_elements=1):
        y8 = torch.nn.functional.linear(x * 1.0, w.detach().half().float())
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(y8, x, dy)[0])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("grad_x", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_lora_layer_with_8_bit_activations(dev, bits, grad_x, p):
    """A LoRALinear's forward and input gradient do not change; dA and dB are the same
    layer's at the held input, bit for bit, and half the memory is kept between."""
    M, K, N = 200, 256, 128
    g = torch.Generator().manual_seed(6)
    layer = LoRALinear(QuantLinear.from_linear(torch.nn.Linear(K, N).to(dev), bits=bits), r=8, lora_dropout=p)
    with torch.no_grad():
        layer.lora_B.copy_(torch.randn(N, 8, generator=g) * 0.1)
    x, dy = torch.randn(M, K, generator=g).to(BF16).to(dev), torch.randn(M, N, generator=g).to(BF16).to(dev)

    def run(x, act_bits):
        layer.activation_bits = act_bits
        x = x.clone().requires_grad_(grad_x)
        torch.manual_seed(1)
        y = layer(x)
        return (y, *torch.autograd.grad(y, ((x,) if grad_x else ()) + (layer.lora_A, layer.lora_B), dy))

    full, held = run(x, 16), run(x, 8)
    for a, b in zip(full[:-2], held[:-2]):
        assert torch.equal(a, b)
    if p == 0.0:
        at = run(decompress(compress(x)), 16)
        assert torch.equal(held[-2], at[-2]) and torch.equal(held[-1], at[-1])
    assert not torch.equal(held[-2], full[-2])
    near = (held[-2] - full[-2]).abs().max() / full[-2].abs().max()
    assert near < 2.0 ** -5  # the held values are within 2^-6 of the block's largest


@pytest.mark.parametrize("M,r", [(200, 8), (8, 8), (96, 96)])
def test_lora_layer_composed_adapter_with_8_bit_activations(dev, M, r):
    """Where the adapter is composed of torch's products (INT8 with fp32 rows, ranks past
    64) the factors and the first product stay as they are: y, dX and dB do not change,
    and dA is the one at the held input."""
    K, N = 96, 64
    g = torch.Generator().manual_seed(8)
    layer = LoRALinear(QuantLinear.from_linear(torch.nn.Linear(K, N).to(dev), bits=8), r=r)
    with torch.no_grad():
        layer.lora_B.copy_(torch.randn(N, r, generator=g) * 0.1)
    x, dy = torch.randn(M, K, generator=g).to(dev), torch.randn(M, N, generator=g).to(dev)

    def run(x, act_bits):
        layer.activation_bits = act_bits
        x = x.clone().requires_grad_(True)
        y = layer(x)
        return (y, *torch.autograd.grad(y, (x, layer.lora_B, layer.lora_A), dy))

    full, held, at = run(x, 16), run(x, 8), run(decompress(compress(x)), 16)
    for a, b in zip(full[:-1], held[:-1]):
        assert torch.equal(a, b)
    assert torch.equal(held[-1], at[-1]) and not torch.equal(held[-1], full[-1])


def test_compiled_layer_runs_its_8_bit_activations_eagerly(dev):
    layer = LoRALinear(QuantLinear.from_linear(torch.nn.Linear(128, 64).to(dev), bits=4), r=8)
    layer.activation_bits = 8
    with torch.no_grad():
        layer.lora_B.normal_()
    x, dy = torch.randn(40, 128, device=dev).to(BF16), torch.randn(40, 64, device=dev).to(BF16)
    torch._dynamo.reset()
    f = torch.compile(lambda x: layer(x * 1.0) * 1.0, backend="eager")
    want = torch.autograd.grad(layer(x), (layer.lora_A, layer.lora_B), dy)
    got = torch.autograd.grad(f(x), (layer.lora_A, layer.lora_B), dy)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(dev):
    with pytest.raises(RuntimeError, match="GPU"):
        compress(torch.zeros(4, 32))
    with pytest.raises(TypeError, match="dtype"):
        compress(torch.zeros(4, 32, dtype=torch.float64, device=dev))
    with pytest.raises(RuntimeError, match="rows expected"):
        compress(torch.zeros((), device=dev))
    with pytest.raises(RuntimeError, match="rows expected"):
        compress(torch.zeros(3, 0, device=dev))
    c, e = ops.act8_quantize(torch.ones(4, 64, device=dev))
    with pytest.raises(RuntimeError, match="not act8_quantize's"):
        ops.act8_dequantize(c, e, 65, FP32)
    with pytest.raises(RuntimeError, match="not act8_quantize's"):
        ops.act8_dequantize(c, e[:, :1], 64, FP32)
