"""ops.mx4_linear's arguments that are about its rows, with the library replaced: no GPU is needed."""
import contextlib

import pytest
import torch

from rocm_qlora import _native as nat
from rocm_qlora import ops


class _Launched(Exception):
    pass


@pytest.fixture
def no_library(monkeypatch):
    def call(name, *args):
        raise _Launched(name)

    monkeypatch.setattr(nat, "require_gpu", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(nat, "call", call)
    monkeypatch.setattr(nat, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(ops, "on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_scratch", lambda fn, dev, *args: None)


def test_rows_are_shared_by_a_plan_alone(no_library):
    x, codes, scales = torch.zeros(4, 64), torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 4, dtype=torch.uint8)
    for M in (None, 4):
        with pytest.raises(_Launched):
            ops.mx4_linear(x, codes, scales, 64, M=M)
    for M in (8, 2, 0):
        with pytest.raises(RuntimeError, match="without a plan"):
            ops.mx4_linear(x, codes, scales, 64, M=M)
    plan = torch.zeros(16, dtype=torch.uint8)
    plan.grouped = (8, 3)
    codes, scales = codes.expand(3, 16, 64).contiguous(), scales.expand(3, 16, 4).contiguous()
    with pytest.raises(_Launched):
        ops.mx4_linear(x, codes, scales, 64, plan=plan, M=8)
    for M in (None, 7, 4):
        with pytest.raises(RuntimeError):
            ops.mx4_linear(x, codes, scales, 64, plan=plan, M=M)
