"""Adapters of many requests, 8-bit checkpoints and the preference loss without a GPU: the
C entry points check their arguments before any HIP call, sizes are what their layouts
need, and tensors off the GPU are refused."""
import ctypes

import pytest
import torch

from rocm_qlora import _native as nat
from rocm_qlora import ops
from rocm_qlora.checkpoint import compress
from rocm_qlora.lora import AdapterRows, MultiLoRALinear, multi_lora
from rocm_qlora.losses import preference_loss, sequence_logps

NULL, DTYPE, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE = 1, 2, 3, 4, 5, 6
A = 4096  # an address that is never read: every call returns before a launch


def raw(name, *args):
    return getattr(nat.load(), name)(*args)


def size(name, *args):
    n = ctypes.c_int64(-1)
    nat.call(name, *args, ctypes.byref(n))
    return n.value


def test_adapter_rows_arguments():
    n = ctypes.c_int64(0)
    assert raw("rq_adapter_rows_size", 8, 4, None) == NULL
    assert raw("rq_adapter_rows_size", -1, 4, ctypes.byref(n)) == SHAPE
    assert raw("rq_adapter_rows_size", 8, 0, ctypes.byref(n)) == SHAPE
    assert raw("rq_adapter_rows_size", 8, ops.MAX_ADAPTERS + 1, ctypes.byref(n)) == UNSUPPORTED
    need = size("rq_adapter_rows_size", 8, 4)
    assert raw("rq_adapter_rows", None, 8, 4, A, need, None) == NULL
    assert raw("rq_adapter_rows", A, 8, 4, None, need, None) == NULL
    assert raw("rq_adapter_rows", A, 8, 4, A, need - 1, None) == WORKSPACE
    assert raw("rq_adapter_rows", A, 8, 4, A + 4, need, None) == ALIGN


@pytest.mark.parametrize("M", [0, 1, 63, 64, 65, 1000, 65536])
@pytest.mark.parametrize("n", [1, 2, 7, 1024])
def test_plan_and_operand_sizes(M, n):
    """A plan holds a slot for every row of the worst grouping: each of min(n + 1, M)
    groups may leave all but one of a tile's 64 slots empty."""
    tiles = M // 64 + min(n + 1, M)
    words = size("rq_adapter_rows_size", M, n) / 4
    assert words >= 16 + 2 * tiles + 64 * tiles + 2 * 4 * (n + 32) + 2 * 2 * n
    for rank, padded in ((1, 16), (16, 16), (17, 32), (33, 64), (512, 512)):
        assert size("rq_multi_lora_u_size", M, n, rank, 1) == 64 * tiles * padded * 4
    assert size("rq_multi_lora_u_size", M, 1, 8, 0) == -(-M // 64) * 64 * 16 * 4


def lora_args(**kw):
    d = dict(x=A, dtype=nat.DTYPE_BF16, M=8, K=32, ldx=32, plan=A, plan_bytes=1 << 20, a=A, b=A, s=A, n=2, rank=4, N=16,
             base=None, ldb=0, out=A, ldo=16, u=None, scratch=A, bytes=1 << 20)
    d.update(kw)
    return (*d.values(), None)


def test_multi_lora_arguments():
    f = lambda **kw: raw("rq_multi_lora", *lora_args(**kw))
    assert f(dtype=9) == DTYPE
    for bad in (dict(K=0), dict(N=0), dict(n=0), dict(rank=0), dict(M=-1), dict(ldx=31), dict(ldo=15), dict(base=A, ldb=15),
                dict(plan_bytes=64)):
        assert f(**bad) == SHAPE, bad
    assert f(n=1025) == UNSUPPORTED and f(rank=513) == UNSUPPORTED
    for null in ("x", "a", "b", "s", "out", "scratch", "plan"):
        assert f(**{null: None}) == NULL, null
    for odd in (dict(x=A + 1), dict(a=A + 1), dict(b=A + 1), dict(out=A + 1), dict(scratch=A + 16), dict(s=A + 2), dict(plan=A + 4),
                dict(base=A + 1, ldb=16), dict(u=A + 4)):
        assert f(**odd) == ALIGN, odd
    assert f(bytes=16) == WORKSPACE
    assert f(M=0) == 0


def grad_args(**kw):
    d = dict(x=A, exps=None, dtype=nat.DTYPE_BF16, M=8, K=32, ldx=32, dy=A, N=16, lddy=16, plan=A, plan_bytes=1 << 20, a=A, b=A,
             s=A, n=2, rank=4, u=A, dxb=None, lddxb=0, dx=A, lddx=32, da=A, db=A, scratch=A, bytes=1 << 24)
    d.update(kw)
    return (*d.values(), None)


def test_multi_lora_grads_arguments():
    f = lambda **kw: raw("rq_multi_lora_grads", *grad_args(**kw))
    assert f(dtype=9) == DTYPE
    for bad in (dict(lddy=15), dict(ldx=31), dict(lddx=31), dict(dxb=A, lddxb=31), dict(exps=A, ldx=40), dict(M=0)):
        assert f(**bad) == SHAPE, bad
    for null in ("x", "dy", "a", "b", "s", "u", "scratch", "plan"):
        assert f(**{null: None}) == NULL, null
    for odd in (dict(dx=A + 1), dict(da=A + 1), dict(db=A + 1), dict(dy=A + 1), dict(u=A + 4), dict(exps=A, x=A + 8)):
        assert f(**odd) == ALIGN, odd
    assert f(bytes=16) == WORKSPACE
    assert f(dx=None, da=None, db=None) == 0


def test_act8_arguments():
    q = lambda *a: raw("rq_act8_quantize", *a, None)
    assert q(A, 9, 2, 32, 32, A, A) == DTYPE
    assert q(A, 0, 2, 0, 32, A, A) == SHAPE and q(A, 0, 2, 32, 31, A, A) == SHAPE and q(A, 0, -1, 32, 32, A, A) == SHAPE
    assert q(A, 0, 1 << 30, 1 << 20, 1 << 20, A, A) == UNSUPPORTED
    assert q(None, 0, 2, 32, 32, A, A) == NULL and q(A, 0, 2, 32, 32, None, A) == NULL and q(A, 0, 2, 32, 32, A, None) == NULL
    assert q(A + 2, 0, 2, 32, 32, A, A) == ALIGN and q(A, 0, 2, 32, 32, A + 8, A) == ALIGN
    assert q(None, 0, 0, 32, 32, None, None) == 0
    d = lambda *a: raw("rq_act8_dequantize", *a, None)
    assert d(A, A, 2, 32, A, 9, 32) == DTYPE and d(A, A, 2, 32, A, 0, 31) == SHAPE and d(A, None, 2, 32, A, 0, 32) == NULL


def test_preference_arguments():
    def f(**kw):
        d = dict(z=A, dtype=nat.DTYPE_F32, T=8, V=16, ld=16, period=0, outer=0, labels=A, offsets=A, S=2, ignore=-100, ref=None,
                 beta=0.1, eps=0.0, average=0, logps=A, loss=A, coef=A, info=A, ws=A, bytes=1 << 20)
        d.update(kw)
        return raw("rq_preference_forward", *d.values(), None)
    assert f(dtype=9) == DTYPE
    for bad in (dict(T=0), dict(V=0), dict(ld=15), dict(S=0), dict(S=3), dict(offsets=None, T=9), dict(period=-1)):
        assert f(**bad) == SHAPE, bad
    for null in ("z", "labels", "logps", "coef", "info", "ws"):
        assert f(**{null: None}) == NULL, null
    assert f(bytes=16) == WORKSPACE and f(ws=A + 16) == ALIGN and f(info=A + 4) == ALIGN and f(z=A + 2) == ALIGN
    b = lambda *a: raw("rq_preference_backward", *a, None)
    assert b(A, 0, 8, 16, 16, 0, 0, A, A, None, 0, A, 15) == SHAPE
    assert b(A, 0, 8, 16, 16, 0, 0, None, A, None, 0, A, 16) == NULL
    assert b(A, 0, 8, 16, 16, 0, 0, A, A, None, 0, A + 2, 16) == ALIGN
    assert b(A, 0, 0, 16, 16, 0, 0, None, None, None, 0, None, 16) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="tensors off the GPU are the case")
def test_tensors_off_the_gpu_are_refused():
    x, a, b = torch.zeros(4, 32), torch.zeros(1, 4, 32), torch.zeros(1, 8, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        AdapterRows(torch.zeros(4, dtype=torch.int32), 1)
    with pytest.raises(RuntimeError, match="GPU"):
        multi_lora(x, a, b, torch.ones(1), AdapterRows.single(4))
    with pytest.raises(RuntimeError, match="GPU"):
        compress(x)
    with pytest.raises(RuntimeError, match="GPU"):
        preference_loss(torch.zeros(2, 4, 8), torch.zeros(2, 4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        sequence_logps(torch.zeros(2, 4, 8, requires_grad=True), torch.zeros(2, 4, dtype=torch.int64))


def test_layer_parameters():
    from rocm_qlora import QuantLinear
    layer = MultiLoRALinear(QuantLinear(64, 32, bits=4), 3, r=4, lora_alpha=8)
    assert layer.lora_A.shape == (3, 4, 64) and layer.lora_B.shape == (3, 32, 4)
    assert not layer.lora_B.any() and bool(layer.lora_A.any()) and layer.scaling.tolist() == [2.0] * 3
    assert {n for n, p in layer.named_parameters() if p.requires_grad} == {"lora_A", "lora_B"}
    with pytest.raises(RuntimeError, match="adapter rows"):
        layer(torch.zeros(2, 64))
