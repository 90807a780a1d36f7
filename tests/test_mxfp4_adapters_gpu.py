"""LoRALinear on a frozen layer that composes its adapter of torch's products (MXFP4Linear): its options do what they
do on a QuantLinear."""
import pytest
import torch

from rocm_qlora import LoRALinear, MXFP4Linear
from rocm_qlora.checkpoint import compress, decompress

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("shape,r", [((200, 96), 8), ((64, 96), 8), ((8, 96), 8), ((96, 96), 96), ((3, 50, 96), 4)])
def test_8_bit_activations(dev, shape, r, p, dtype):
    """y, dX and dB do not change, dA is the one at the held input (a batch of as many rows as the factors have, or the
    weight, among the shapes)."""
    K, N = shape[-1], 64
    g = torch.Generator().manual_seed(8)
    layer = LoRALinear(MXFP4Linear.from_linear(torch.nn.Linear(K, N).to(dev)), r=r, lora_dropout=p)
    with torch.no_grad():
        layer.lora_B.copy_(torch.randn(N, r, generator=g) * 0.1)
    x, dy = torch.randn(shape, generator=g).to(dtype).to(dev), torch.randn(*shape[:-1], N, generator=g).to(dtype).to(dev)

    def run(x, bits):
        layer.activation_bits = bits
        x = x.clone().requires_grad_(True)
        torch.manual_seed(1)
        y = layer(x)
        return (y, *torch.autograd.grad(y, (x, layer.lora_B, layer.lora_A), dy))

    full, held = run(x, 16), run(x, 8)
    for a, b in zip(full[:-1], held[:-1]):
        assert torch.equal(a, b)
    assert not torch.equal(held[-1], full[-1])
    if p == 0.0:
        assert torch.equal(held[-1], run(decompress(compress(x)), 16)[-1])
    # without a gradient nothing is held
    with torch.no_grad():
        layer.activation_bits = 8
        torch.manual_seed(1)
        assert torch.equal(layer(x), full[0])


def test_8_bit_activations_keep_half_the_memory(dev):
    M, K, N = 4096, 4096, 256
    layer = LoRALinear(MXFP4Linear(K, N).to(dev), r=8)
    x = torch.randn(M, K, device=dev).to(BF16)

    def kept(bits):
        layer.activation_bits = bits
        h = x * 1.0  # an activation of the layer's own
        before = torch.cuda.memory_allocated()
        y = layer(h)
        del h
        return torch.cuda.memory_allocated() - before, y

    full, _ = kept(16)
    held, _ = kept(8)
    assert held < full - M * K * 2 * 0.4
