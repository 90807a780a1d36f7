"""What 8-bit activations leave as it is: parameters by whatever view or cast, and a layer's
factors where they have its input's shape."""
import pytest
import torch

from rocm_qlora import LoRALinear, QuantLinear
from rocm_qlora.checkpoint import compress, decompress, saved_in_8_bits

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16

VIEWS = {
    "rows": lambda p: p[8:72],
    "columns": lambda p: p[:, 16:],
    "one of several": lambda p: p.view(2, 40, 96)[1],
    "unbound": lambda p: p.view(2, 40, 96).unbind(0)[0],
    "split": lambda p: p.split(40)[1],
    "sized split": lambda p: p.split([30, 50])[1],
    "chunk": lambda p: p.chunk(2, 1)[0],
    "unsqueezed": lambda p: p.unsqueeze(0).squeeze(0),
    "expanded": lambda p: p[:1].expand(40, 96),
    "transposed copy": lambda p: p.t().contiguous().t(),
    "cast of a slice": lambda p: p[:40].to(BF16).float(),
    "slice of a cast": lambda p: p.to(BF16).float()[:40],
    "movedim": lambda p: p.view(2, 40, 96).movedim(0, 1)[:, 0],
}


@pytest.mark.parametrize("view", list(VIEWS))
def test_views_of_parameters_stay_as_they_are(dev, view):
    """The input gradient of a linear is dY W: with W any view, copy or cast of a parameter it
    does not change, and the weight's gradient is the one at the held input."""
    g = torch.Generator().manual_seed(4)
    p = torch.nn.Parameter(torch.randn(80, 96, generator=g).to(dev))
    w = VIEWS[view](p)
    x = torch.randn(64, w.shape[1], generator=g).to(dev).requires_grad_(True)
    dy = torch.randn(64, w.shape[0], generator=g).to(dev)

    def grads(bits):
        h = x * 1.0
        if bits == 8:
            with saved_in_8_bits(min_elements=1):
                y = torch.nn.functional.linear(h, w)
        else:
            y = torch.nn.functional.linear(h, w)
        return (y, *torch.autograd.grad(y, (x, p), dy, retain_graph=True))

    (y0, dx0, dp0), (y8, dx8, dp8) = grads(16), grads(8)
    assert torch.equal(y0, y8) and torch.equal(dx0, dx8)
    assert not torch.equal(dp0, dp8)  # the input itself is held in 8 bits


def test_factors_of_the_inputs_shape_stay_as_they_are(dev):
    """A batch of as many rows as ranks, factors that are no parameters (functional_call): A has
    x's shape.  y, dX and dB do not change, dA and dB are those at the held input."""
    K, N, r = 128, 64, 8
    g = torch.Generator().manual_seed(8)
    layer = LoRALinear(QuantLinear.from_linear(torch.nn.Linear(K, N).to(dev), bits=4), r=r)
    factors = {"lora_A": torch.randn(r, K, generator=g).to(BF16).to(dev), "lora_B": torch.randn(N, r, generator=g).to(BF16).to(dev)}
    x, dy = torch.randn(r, K, generator=g).to(BF16).to(dev), torch.randn(r, N, generator=g).to(BF16).to(dev)

    def run(x, bits):
        layer.activation_bits = bits
        x = x.clone().requires_grad_(True)
        f = {k: v.clone().requires_grad_(True) for k, v in factors.items()}
        y = torch.func.functional_call(layer, f, (x,))
        return (y, *torch.autograd.grad(y, (x, f["lora_A"], f["lora_B"]), dy))

    full, held, at = run(x, 16), run(x, 8), run(decompress(compress(x)), 16)
    assert torch.equal(held[0], full[0]) and torch.equal(held[1], full[1])
    assert torch.equal(held[2], at[2]) and torch.equal(held[3], at[3]) and not torch.equal(held[2], full[2])


@pytest.mark.parametrize("cast", [False, True])
def test_frozen_factors_of_the_inputs_shape_stay_as_they_are(dev, cast):
    """The composed adapter of a square layer (INT8 with fp32 rows) whose B is frozen: B's
    transpose, or its cast's, has the shape of a batch of as many rows as ranks."""
    K, r = 96, 16
    g = torch.Generator().manual_seed(9)
    layer = LoRALinear(QuantLinear.from_linear(torch.nn.Linear(K, K).to(dev), bits=8), r=r)
    with torch.no_grad():
        layer.lora_B.copy_(torch.randn(K, r, generator=g) * 0.1)
    if cast:
        layer.lora_B.data = layer.lora_B.data.to(BF16)
    layer.lora_B.requires_grad_(False)
    x, dy = torch.randn(r, K, generator=g).to(dev), torch.randn(r, K, generator=g).to(dev)

    def run(x, bits):
        layer.activation_bits = bits
        x = x.clone().requires_grad_(True)
        y = layer(x)
        return (y, *torch.autograd.grad(y, (x, layer.lora_A), dy))

    full, held, at = run(x, 16), run(x, 8), run(decompress(compress(x)), 16)
    assert torch.equal(held[0], full[0]) and torch.equal(held[1], full[1])
    assert torch.equal(held[2], at[2]) and not torch.equal(held[2], full[2])
