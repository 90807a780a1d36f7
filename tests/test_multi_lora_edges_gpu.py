"""Adapters of many requests where tiles, ranks and magnitudes end: bounds and oracle are
test_multi_lora_gpu.py's."""
import pytest
import torch

from rocm_qlora.lora import AdapterRows
from test_multi_lora_gpu import BF16, E32, FP16, FP32, U, check_all, make, oracle, run_all

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("r", [80, 96, 160, 224, 352])
@pytest.mark.parametrize("M,bits", [(64, 16), (192, 16), (128, 8)])
def test_ranks_that_leave_a_wave_part_of_its_blocks(dev, M, bits, r, dtype):
    """Padded ranks past 64 that are no multiple of 64, in tiles that are full, so that the
    operands end with their buffer: without grouping and grouped."""
    print(f"multi_lora r={r} M={M} {dtype} bits={bits}", flush=True)
    d = make(M, 96, 72, r, 1, dtype, dev, seed=r, ids=torch.zeros(M))
    check_all(d, run_all(d, AdapterRows.single(M), bits), bits)
    d = make(M, 96, 72, r, 2, dtype, dev, seed=r + 1, ids=[m // 64 % 2 for m in range(M)])
    check_all(d, run_all(d, AdapterRows(d["ids"], 2), bits), bits)


@pytest.mark.parametrize("M", [6, 30, 192])
@pytest.mark.parametrize("r", [5, 16, 40, 96])
@pytest.mark.parametrize("small", ["a", "b"])
def test_small_first_products_in_fp16(dev, M, r, small):
    """fp16 factors at a training's start: first products of 1e-6 (x A^T where A is small,
    dY B where B is), results of ordinary size by the scaling.  A first product's two parts
    hold 22 bits of it, and 2^-36 where that is more: no result loses more than that times
    the second product's other operand, beside its own rounding (2^-25 below 2^-14)."""
    print(f"small {small} M={M} r={r}", flush=True)
    d = make(M, 64, 8, r, 1, FP16, dev, seed=r + M, ids=torch.zeros(M))
    s = 2.0 ** 12
    d["base"].zero_()
    d["s"].fill_(s)
    if small == "a":
        d["a"], d["dy"] = d["a"] * 2.0 ** -18, d["dy"] * 2.0 ** -3
    else:
        d["b"], d["dy"] = d["b"] * 2.0 ** -12, d["dy"] * 2.0 ** -5
    got = run_all(d, AdapterRows.single(M))
    want, absum, step = oracle(d)
    first = (d["x"].double() @ d["a"][0].double().T) if small == "a" else (d["dy"].double() @ d["b"][0].double())
    assert 2.0 ** -24 < first.abs().mean().item() < 2.0 ** -14
    (M, K), N = d["x"].shape, 8
    for i, name in ((0, "y"), (3, "dB")) if small == "a" else ((1, "dx"), (2, "dA")):
        other = step[i] * (s if name in ("dx", "dA") else 1.0)  # the oracle's steps of y and dB have the scaling
        bound = U[FP16] * want[i].abs() + (U[FP16] ** 2 + (K + N + M + r + 8) * E32) * absum[i] + 2.0 ** -36 * other + 2.0 ** -25
        worst = ((got[i].double().cpu() - want[i]).abs() / bound).max().item()
        assert worst <= 1.0, f"{name}: error {worst:.2f} times its bound"
