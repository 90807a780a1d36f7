"""The MXFP4 linears without a GPU: the C entry points check their arguments before any HIP call,
modules hold what they document, and calls that are not supported are refused."""
import ctypes

import numpy as np
import pytest
import torch

import mxfp4_oracle as oracle
from rocm_qlora import (ExpertRows, LoRALinear, MXFP4Experts, MXFP4Linear, MXFP4Tensor, dequantize_mxfp4, mxfp4_expert_linear,
                        mxfp4_linear, ops, quantize_mxfp4)
from rocm_qlora import _native as nat
from rocm_qlora.export.gguf_export import merge_and_export_fp16
from rocm_qlora.lora import MultiLoRALinear

NULL, DTYPE, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE = 1, 2, 3, 4, 5, 6
A = 4096  # an address that is never read: every call returns before a launch


def raw(name, *args):
    return getattr(nat.load(), name)(*args)


def size(name, *args):
    n = ctypes.c_int64(-1)
    nat.call(name, *args, ctypes.byref(n))
    return n.value


def test_codec_arguments():
    q = lambda *a: raw("rq_mx4_quantize", *a, None)
    assert q(A, 9, 2, 32, 32, A, A) == DTYPE
    assert q(A, 0, 2, 0, 32, A, A) == SHAPE and q(A, 0, 2, 32, 31, A, A) == SHAPE and q(A, 0, -1, 32, 32, A, A) == SHAPE
    assert q(A, 0, 1 << 30, 1 << 20, 1 << 20, A, A) == UNSUPPORTED
    for i in (0, 5, 6):
        args = [A, 0, 2, 32, 32, A, A]
        args[i] = None
        assert q(*args) == NULL
    assert q(A + 2, 0, 2, 32, 32, A, A) == ALIGN and q(A, 0, 2, 32, 32, A + 8, A) == ALIGN
    assert q(None, 0, 0, 32, 32, None, None) == 0
    d = lambda *a: raw("rq_mx4_dequantize", *a, None)
    assert d(A, A, 2, 32, A, 9, 32) == DTYPE
    assert d(A, A, 2, 32, A, 0, 31) == SHAPE and d(A, A, 2, 0, A, 0, 31) == SHAPE
    assert d(None, A, 2, 32, A, 0, 32) == NULL and d(A, None, 2, 32, A, 0, 32) == NULL and d(A, A, 2, 32, None, 0, 32) == NULL
    assert d(A + 8, A, 2, 32, A, 0, 32) == ALIGN and d(A, A, 2, 32, A + 2, 0, 32) == ALIGN
    assert d(None, None, 0, 32, None, 0, 32) == 0


def linear(**kw):
    d = dict(x=A, dtype=nat.DTYPE_BF16, M=8, K=64, ldx=64, shared=1, plan=None, plan_bytes=0, codes=A, scales=A, E=1, N=16, bias=None,
             bits=16, y=A, ldy=16, scratch=None, bytes=0)
    d.update(kw)
    return raw("rq_mx4_linear", *d.values(), None)


def linear_dx(**kw):
    d = dict(dy=A, dtype=nat.DTYPE_BF16, M=8, N=16, lddy=16, plan=None, plan_bytes=0, codes=A, scales=A, E=1, K=64, shared=1, dx=A,
             lddx=64, scratch=None, bytes=0)
    d.update(kw)
    return raw("rq_mx4_linear_dx", *d.values(), None)


def test_linear_arguments():
    for f, inp, out in ((linear, "x", "y"), (linear_dx, "dy", "dx")):
        assert f(dtype=9) == DTYPE
        for bad in (dict(M=-1), dict(K=0), dict(N=0), dict(E=0), dict(E=2), dict(shared=0), dict(shared=2), {f"ld{inp}": 15},
                    {f"ld{out}": 15}, dict(plan=A, shared=3)):
            assert f(**bad) == SHAPE, bad
        for far in (dict(plan=A, E=ops.MAX_ADAPTERS + 1), dict(M=1 << 31), dict(K=1 << 25, ldx=1 << 25) if f is linear else dict(K=1 << 25),
                    dict(N=1 << 31), dict(K=1 << 20, N=1 << 16)):
            assert f(**far) == UNSUPPORTED, far
        for null in (inp, out, "codes", "scales"):
            assert f(**{null: None}) == NULL, null
        for odd in ({inp: A + 1}, {out: A + 1}, dict(codes=A + 8), dict(scales=A + 2), dict(plan=A + 4, plan_bytes=1 << 20)):
            assert f(**odd) == ALIGN, odd
        assert f(plan=A, plan_bytes=64) == WORKSPACE
        assert f(M=0, **{inp: None, out: None}) == 0
    assert linear(bias=A + 1) == ALIGN
    assert linear(bits=8) == UNSUPPORTED and linear(bits=4, plan=A) == UNSUPPORTED


def test_scratch_size_arguments():
    n = ctypes.c_int64(-1)
    f = lambda *a: raw("rq_mx4_linear_scratch_size", *a, ctypes.byref(n))
    assert raw("rq_mx4_linear_scratch_size", 1, 8, 64, 16, 1, 1, 0, 16, 0, 64, 1, None) == NULL
    assert f(9, 8, 64, 16, 1, 1, 0, 16, 0, 64, 1) == DTYPE
    assert f(1, 8, 64, 16, 1, 1, 0, 16, 0, 63, 1) == SHAPE and f(1, 8, 64, 16, 1, 1, 0, 16, 1, 15, 1) == SHAPE
    assert f(1, 8, 64, 16, 2, 1, 0, 16, 0, 64, 1) == SHAPE and f(1, 9, 64, 16, 2, 2, 1, 16, 0, 64, 1) == SHAPE
    assert f(1, 8, 64, 16, 2, 1, 1, 4, 0, 64, 1) == UNSUPPORTED
    assert f(1, 0, 64, 16, 1, 1, 0, 16, 0, 64, 1) == 0 and n.value == 0


@pytest.mark.parametrize("M,n", [(0, 1), (1, 1024), (65, 3), (4096, 8)])
def test_a_plan_holds_the_tables_of_larger_tiles(M, n):
    """Of two and of four 64-row tiles: one entry each for every group's, whole or not."""
    tiles = M // 64 + min(n + 1, M)
    base = 16 + 2 * tiles + 64 * tiles + 2 * 4 * (n + 32) + 2 * 2 * n
    most = sum(M // (64 * m) + min(n + 1, M) for m in (2, 4))
    assert size("rq_adapter_rows_size", M, n) / 4 >= base + most


def tensor(N, K, lead=()):
    return MXFP4Tensor(torch.zeros(*lead, N, ops.mx4_pad(K) // 2, dtype=torch.uint8),
                       torch.zeros(*lead, N, ops.mx4_pad(K) // 32, dtype=torch.uint8), K)


def test_tensor_and_modules():
    t = tensor(5, 130, (2,))
    assert t.shape == (2, 5, 130) and t.nbytes() == 2 * 5 * (128 + 8) and "2, 5, 130" in repr(t)
    assert t.to("cpu").shape == t.shape
    c, s = t.codes, t.scales
    for bad in ((c, s, 0), (c, s, 257), (c, s, 128), (c[:1], s, 130), (c, s[..., :4], 130), (c[..., ::2], s[..., ::2], 128),
                (c.transpose(0, 1), s.transpose(0, 1), 130)):
        with pytest.raises(RuntimeError, match="MXFP4"):
            MXFP4Tensor(*bad)
    with pytest.raises(TypeError, match="uint8"):
        MXFP4Tensor(c.to(torch.int8), s, 130)
    m = MXFP4Linear(130, 5, activation_bits=4)
    assert set(m.state_dict()) == {"weight_quant", "weight_scales", "bias"} and not m.bias.requires_grad
    assert "in_features=130" in repr(m) and "activation_bits=4" in repr(m)
    # codes and scales keep their type when a module changes its own
    assert m.half().weight_quant.dtype == torch.uint8 and m.bias.dtype == torch.half
    e = MXFP4Experts(3, 130, 5)
    assert e.weight_quant.shape == (3, 5, 128) and e.weight_scales.shape == (3, 5, 8) and e.bias is None and "n=3" in repr(e)
    with pytest.raises(ValueError, match="activation_bits"):
        MXFP4Linear(130, 5, activation_bits=8)


def test_layers_beside_it_refuse_what_it_cannot_do(tmp_path):
    lora = LoRALinear(MXFP4Linear(64, 32), r=4)
    assert [n for n, p in lora.named_parameters() if p.requires_grad] == ["lora_A", "lora_B"]
    with pytest.raises(TypeError, match="MXFP4Linear"):
        lora.merge_lora()
    assert not lora.merged
    with pytest.raises(TypeError, match="MXFP4Linear"):
        merge_and_export_fp16(torch.nn.Sequential(lora), str(tmp_path / "w.pt"))
    with pytest.raises(TypeError, match="MXFP4Linear"):
        MultiLoRALinear(MXFP4Linear(64, 32), 2)


def test_experts_weights_that_differ_are_refused():
    for bad in ([], [torch.nn.Linear(8, 4), torch.nn.Linear(8, 4, bias=False)], [torch.nn.Linear(8, 4), torch.nn.Linear(8, 5)],
                torch.zeros(0, 4, 8)):
        with pytest.raises(ValueError):
            MXFP4Experts.from_weights(bad)
    with pytest.raises(RuntimeError, match="experts"):
        MXFP4Experts.from_weights(torch.zeros(4, 8))


@pytest.mark.skipif(torch.cuda.is_available(), reason="tensors off the GPU are the case")
def test_tensors_off_the_gpu_are_refused():
    x, w = torch.zeros(4, 64), tensor(16, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        mxfp4_linear(x, w)
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_mxfp4(x)
    with pytest.raises(RuntimeError, match="GPU"):
        dequantize_mxfp4(w)
    with pytest.raises(RuntimeError, match="GPU"):
        ExpertRows(torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.mx4_linear_dx(torch.zeros(4, 16), w.codes, w.scales, 64)


def test_calls_that_do_not_fit_are_refused():
    x, w = torch.zeros(4, 64), tensor(16, 64)
    for bad in (torch.zeros(()), torch.zeros(4, 65)):
        with pytest.raises(RuntimeError, match="rows of 64"):
            mxfp4_linear(bad, w)
    with pytest.raises(RuntimeError, match="gradient by bias"):
        mxfp4_linear(x, w, torch.zeros(16, requires_grad=True))
    for ids in (torch.zeros((), dtype=torch.int32), torch.zeros(2, 2, 2, dtype=torch.int32), torch.zeros(4, 0, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="ids"):
            ExpertRows(ids, 2)
    rows = ExpertRows.__new__(ExpertRows)
    rows.M, rows.n, rows.k, rows.plan = 8, 2, 2, torch.zeros(16, dtype=torch.uint8)
    we = tensor(16, 64, (2,))
    for bad in (torch.zeros(3, 64), torch.zeros(4, 63), torch.zeros(2, 4, 64)):
        with pytest.raises(RuntimeError, match="x must be"):
            mxfp4_expert_linear(bad, we, rows)
    for bad in (w, tensor(16, 64, (3,))):
        with pytest.raises(RuntimeError, match="2 experts"):
            mxfp4_expert_linear(x, bad, rows)


def test_plans_of_other_rows_are_refused():
    """Also where the sizes are the same."""
    plan = torch.zeros(16, dtype=torch.uint8)
    plan.grouped = (16, 3)
    ops._mx4_plan(plan, 16, 3)
    for p, M, E in ((plan, 8, 3), (plan, 16, 4), (plan.clone(), 16, 3)):
        with pytest.raises(RuntimeError, match="by expert"):
            ops._mx4_plan(p, M, E)


def test_the_oracle_against_the_format():
    """Every code and many scales by hand: the oracle's values are what the format defines, and quantizing them
    again gives them back."""
    codes = torch.arange(16).repeat(8)[None].numpy()
    scales = np.array([[1, 100, 127, 200]])
    v = oracle.values(codes, scales)
    grid = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    for b, e in enumerate((1, 100, 127, 200)):
        assert v[0, 32 * b:32 * b + 16].tolist() == [s * g * 2.0 ** (e - 127) for s in (1, -1) for g in grid]
    c, s, back = oracle.quantize(torch.from_numpy(v))
    assert (back == v).all() and (s == scales).all() and (c[v != 0] == codes[v != 0]).all()
