"""The rows by adapter that ops.multi_lora and its gradients take: those that adapter_rows made for as many rows and
adapters, whatever their size.  The library is replaced, so no GPU is needed."""
import contextlib
import copy
import ctypes
import pickle

import pytest
import torch

from rocm_qlora import _native as nat
from rocm_qlora import ops

K, N, R = 64, 48, 4


class _Launched(Exception):
    pass


def size(M, n):
    out = ctypes.c_int64(-1)
    assert nat.load().rq_adapter_rows_size(M, n, ctypes.byref(out)) == 0
    return out.value


@pytest.fixture
def no_library(monkeypatch):
    def call(name, *args):
        if name in ("rq_multi_lora", "rq_multi_lora_grads"):
            raise _Launched(name)

    sizes = {"rq_adapter_rows_size": size}
    monkeypatch.setattr(nat, "require_gpu", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(nat, "call", call)
    monkeypatch.setattr(nat, "stream_handle", lambda dev: 0)
    monkeypatch.setattr(ops, "on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_bytes", lambda fn, dev, *args: sizes[fn](*args) if fn in sizes else 64)
    monkeypatch.setattr(ops, "_scratch", lambda fn, dev, *args: torch.zeros(sizes[fn](*args) if fn in sizes else 64, dtype=torch.uint8))


def operands(M, n):
    return torch.zeros(M, K), torch.zeros(n, R, K), torch.zeros(n, N, R), torch.ones(n)


def plan(M, n):
    return ops.adapter_rows(torch.zeros(M, dtype=torch.int32), n)


def calls(M, n, p):
    x, a, b, s = operands(M, n)
    u = torch.zeros(64, dtype=torch.uint8)
    real = torch.empty
    yield lambda: ops.multi_lora(x, a, b, s, p, out=real(M, N))
    yield lambda: ops.multi_lora_grads(x, torch.zeros(M, N), a, b, s, p, u)


@pytest.mark.parametrize("M,n", [(8, 2), (100, 3), (65, 1)])
def test_a_plan_of_these_rows_is_taken(no_library, M, n):
    p = plan(M, n)
    for q in (p, copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        for f in calls(M, n, q):
            with pytest.raises(_Launched):
                f()


@pytest.mark.parametrize("M,n,M2,n2", [(127, 3, 65, 3), (65, 3, 127, 3), (200, 2, 192, 2), (8, 2, 7, 2), (64, 3, 64, 2)])
def test_a_plan_of_other_rows_is_refused(no_library, M, n, M2, n2):
    """All but the last have the size of those that are asked for."""
    p = plan(M2, n2)
    assert (p.numel() == size(M, n)) == (n2 == n)
    for f in calls(M, n, p):
        with pytest.raises(RuntimeError, match="rows by adapter are not those"):
            f()
    for f in calls(M, n, plan(M, n).clone()):  # bytes of unknown origin
        with pytest.raises(RuntimeError, match="rows by adapter are not those"):
            f()


def test_several_adapters_need_a_plan(no_library):
    for f in calls(8, 2, None):
        with pytest.raises(RuntimeError, match="without the batch's rows"):
            f()
