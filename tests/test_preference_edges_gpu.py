"""Preference loss where magnitudes end: oracle and bounds are test_preference_gpu.py's.

Near a maximum m the exponent's argument is off by half an ulp of m log2 e, 2^6 at most where
its neighbours count (up to 2^30), and rounded to fp32: 2^-18 of a base-2 logarithm at most,
within the 70 2^-24 that the bound gives a row.  Past 2^30 fp32 values are 128 apart or more,
and e^-128 is no fp32 number: only what equals the maximum counts."""
import pytest
import torch

from rocm_qlora.losses import preference_loss, sequence_logps
from test_preference_gpu import BF16, FP32, check_dz, check_logps, oracle

pytestmark = pytest.mark.gpu


def check_sequences(z, labels, offsets, V, dtype):
    up = torch.linspace(0.5, 2.0, offsets.numel() - 1, device=z.device)
    z = z.clone().requires_grad_(True)
    lp = sequence_logps(z, labels, offsets)
    _, wp, wz, counts = oracle(z, labels, offsets, pairs=False, up=up)
    assert bool(torch.isfinite(wp).all())
    check_logps(lp, wp, counts, V, False)
    check_dz(torch.autograd.grad(lp, z, up)[0], wz, z, dtype, V)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("V", [9, 3000, 100003])
@pytest.mark.parametrize("m", [1e3, 3e7, 5e8, 1e9, 2.0 ** 30, 1e10, 1e20, 1e30, 3e38])
def test_large_finite_maxima(dev, m, V, dtype):
    """Rows of one value, m or -m (a mask's value throughout), and rows that one logit of m
    or of -m leads: log_softmax of all of them is finite."""
    z = torch.zeros(8, V, dtype=dtype, device=dev)
    z[0], z[2] = m, -m          # constant: -log V
    z[4, V - 1] = m             # its logit leads: 0
    z[6] = -torch.finfo(dtype).max if m > 1e30 else -2 * m
    z[6, 3] = -m                # the label is the largest of lower ones: 0
    labels = torch.full((8,), -100, device=dev)
    labels[1], labels[3], labels[5], labels[7] = V // 2, 2, V - 1, 3
    check_sequences(z, labels, torch.arange(0, 9, 2, device=dev), V, dtype)


def test_close_logits_below_a_large_maximum(dev):
    """Neighbours of a large maximum that still count, and those that no longer do."""
    V, at = 40, (2.0 ** 20, 2.0 ** 26, 2.0 ** 29, 2.0 ** 30, 2.0 ** 31)
    z = torch.zeros(2 * len(at), V, device=dev)
    labels = torch.full((2 * len(at),), -100, device=dev)
    for i, m in enumerate(at):
        for sign, cols in ((1.0, range(0, 20)), (1.0, range(20, 40))):
            for v in cols:
                z[2 * i, v] = sign * torch.nextafter(torch.tensor(m), torch.tensor(0.0)) if v % 3 else sign * m
        labels[2 * i + 1] = 3
    check_sequences(z, labels, torch.arange(0, 2 * len(at) + 1, 2, device=dev), V, FP32)
    # the label a neighbour's step below the maximum
    labels[1::2] = 4
    check_sequences(z, labels, torch.arange(0, 2 * len(at) + 1, 2, device=dev), V, FP32)


def test_infinite_ratio_without_smoothing(dev):
    """A rejected answer that the model cannot give (its token masked to -inf): D is +inf, and
    without label smoothing its pair's loss is 0, with it +inf; the other pair counts as it does."""
    z = torch.randn(8, 12, generator=torch.Generator().manual_seed(0)).to(dev)
    labels = torch.tensor([-100, 3] * 4, device=dev)
    offsets = torch.tensor([0, 2, 4, 6, 8], device=dev)
    z[4, 3] = float("-inf")     # sequence 2, the rejected one of pair 0
    z.requires_grad_(True)
    loss, logps = preference_loss(z, labels, offsets)
    other = preference_loss(z[[2, 3, 6, 7]], labels[:4], offsets[:3])[0]
    assert logps[2].item() == float("-inf")
    assert abs(loss.item() - other.item() / 2) <= 2.0 ** -23 * other.item()
    dz = torch.autograd.grad(loss, z)[0]
    assert not dz[0].any() and not dz[4].any() and bool(dz[2].any()) and bool(torch.isfinite(dz).all())
    assert preference_loss(z, labels, offsets, label_smoothing=0.1)[0].item() == float("inf")
    # the chosen one: D is -inf, and all smoothing leaves nothing of it
    z = z.detach().roll(-4, 0)
    assert preference_loss(z, labels, offsets)[0].item() == float("inf")
    all_smooth = preference_loss(z, labels, offsets, label_smoothing=1.0)[0].item()
    assert abs(all_smooth - preference_loss(z[[2, 3, 6, 7]], labels[:4], offsets[:3], label_smoothing=1.0)[0].item() / 2) <= 2.0 ** -23
