"""Adapters of many requests where tiles, ranks and magnitudes end: bounds and oracle are
test_multi_lora_gpu.py's."""
import pytest
import torch

from rocm_qlora.lora import AdapterRows
from test_multi_lora_gpu import BF16, FP16, FP32, check_all, make, run_all

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
