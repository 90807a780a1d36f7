"""MXFP4 weights: codec, linears, and linears of experts (no counterpart in the
reference).

32 consecutive values of a row share a power of two; each is one of 0, 1/2, 1, 3/2,
2, 3, 4, 6 times it, with a sign (the OCP microscaling format MXFP4): 4.25 bits a
value.  With e = floor(log2 max |x|) - 2 of the block, a value's code is the nearest to
x 2^-e, ties to the even code, past 6 it is 6.  A block with an infinity or a NaN
stands for NaN.  gfx950 converts such codes to bf16 in its own instructions and
multiplies them in its scaled matrix instructions, which NF4's table of values cannot
be: the linears here read a weight at 17/32 of a byte a value and decode it in registers.

A frozen base in MXFP4 trains adapters like an NF4 one: forward and input gradient run
on the 4-bit weight, the weight itself has no gradient.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn as nn

from rocm_qlora import ops
from rocm_qlora._device import to_gpu
from rocm_qlora.kernels import dequant_matmul as dm
from rocm_qlora.torch_ops import eager_only, first_order


class MXFP4Tensor:
    """A tensor [..., K] held in MXFP4: codes [..., Kp / 2] and scales [..., Kp / 32] (uint8,
    contiguous; Kp = K rounded up to 128, zero codes after K), two codes a byte with the
    even value in the low bits, scales as exponent + 127."""
    __slots__ = ("codes", "scales", "K")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, K: int):
        ops._check_mx4(codes, scales, K)
        self.codes, self.scales, self.K = codes, scales, int(K)

    @classmethod
    def _of(cls, codes: torch.Tensor, scales: torch.Tensor, K: int) -> "MXFP4Tensor":
        """Of codes and scales that fit."""
        t = cls.__new__(cls)
        t.codes, t.scales, t.K = codes, scales, K
        return t

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.K))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, device) -> "MXFP4Tensor":
        return MXFP4Tensor(self.codes.to(device), self.scales.to(device), self.K)

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={tuple(self.shape)}, device={self.device})"


@eager_only
def quantize_mxfp4(tensor: torch.Tensor) -> MXFP4Tensor:
    """tensor ([..., K] fp32/bf16/fp16) in MXFP4 blocks along its last dimension.  A CPU tensor
    is staged through the GPU and its codes are returned on the CPU, as quantize_int4's."""
    if tensor.is_cuda:
        codes, scales = ops.mx4_quantize(tensor)
    else:
        src, home = to_gpu(tensor.detach())
        codes, scales = (t.to(home) for t in ops.mx4_quantize(src))
    return MXFP4Tensor._of(codes, scales, tensor.shape[-1])


@eager_only
def dequantize_mxfp4(t: MXFP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of t in `dtype` (exact in bf16 and fp32; in fp16 where it holds them)."""
    if t.codes.is_cuda:
        return ops._mx4_dequantize(t.codes, t.scales, t.K, dtype)
    codes, home = to_gpu(t.codes)
    return ops._mx4_dequantize(codes, t.scales.to(codes.device), t.K, dtype).to(home)


class ExpertRows:
    """The rows of a batch grouped by expert, for every projection that they pass through.
    ids: [T] or [T, k] int32 or int64 on the GPU, the experts 0 .. n - 1 of T tokens, or anything
    else for a place without one; made on the current stream, without a host synchronization.  Row t k + j
    is token t's place j."""
    __slots__ = ("M", "n", "k", "plan")

    def __init__(self, ids: torch.Tensor, n: int):
        if ids.dim() not in (1, 2):
            raise RuntimeError(f"ids are [tokens] or [tokens, experts of a token], got {tuple(ids.shape)}")
        if ids.dim() == 2 and ids.shape[1] == 0:
            raise RuntimeError("ids name at least one expert a token")
        self.M, self.n = ids.numel(), int(n)
        self.k = 1 if ids.dim() == 1 else ids.shape[1]
        self.plan = ops.adapter_rows(ids.reshape(-1), self.n)


def _versions(codes: torch.Tensor, scales: torch.Tensor):
    """How often each has been written to in place (inference tensors do not count that)."""
    return -1 if codes.is_inference() else codes._version, -1 if scales.is_inference() else scales._version


class _MXFP4Linear(torch.autograd.Function):
    """y by the linears' kernels, dX in the backward pass.  w: a weight's (codes, scales, K), frozen: kept as
    it is, not among autograd's saved tensors, whose hooks (8-bit checkpoints, offloading) are for activations.  As
    for those, a write to it in between is refused."""

    @staticmethod
    def forward(ctx, x, w, bias, bits, rows):
        codes, scales, K = w
        ctx.versions = _versions(codes, scales)
        if rows is None:
            ctx.args = (codes, scales, K, 1, codes.shape[0], None, 1)
            return ops._mx4_linear(x, codes, scales, K, bias, bits, None, None)
        R = x.shape[0]
        ctx.args = (codes, scales, K, codes.shape[0], codes.shape[1], rows.plan, rows.M // R if R else 1)
        return ops._mx4_linear(x, codes, scales, K, bias, bits, rows.plan, rows.M)

    @staticmethod
    @first_order
    def backward(ctx, dy):
        if _versions(*ctx.args[:2]) != ctx.versions:
            raise RuntimeError("the MXFP4 weight needed for gradient computation has been modified by an inplace operation "
                               "since the forward pass")
        return ops._mx4_dx(dy, *ctx.args), None, None, None, None


def _refuse_bias_gradient(bias: Optional[torch.Tensor], name: str) -> None:
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} has no gradient by bias: pass it detached")


def _linear(x, codes, scales, K, bias, bits):
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    if dm._nothing_recorded_eagerly(x):
        y = ops._mx4_linear(x2, codes, scales, K, bias, bits, None, None)
    else:
        y = _MXFP4Linear.apply(x2, (codes, scales, K), bias, bits, None)
    return y if flat else y.view(*x.shape[:-1], y.shape[-1])


@eager_only
def mxfp4_linear(x: torch.Tensor, w: MXFP4Tensor, bias: Optional[torch.Tensor] = None, activation_bits: int = 16) -> torch.Tensor:
    """x w^T + bias for a weight [N, K] in MXFP4.

    x: [..., K] fp32, bf16 or fp16 on the GPU; the result has its dtype.  The weight's values are
    exact beside bf16 and fp32 rows, and rounded to fp16 beside fp16 rows (exact for scales of 2^-23 ..
    2^13); sums are fp32, bias is added to them (in x's dtype) and the result rounded once.  fp32 rows
    are multiplied as three bf16 parts each, which hold all their bits.
    activation_bits=4: x's rows are quantized as quantize_mxfp4 does first, and codes multiplied by codes.
    Differentiable by x: dX = dY w (activation_bits=4: as if x had not been rounded), once."""
    if bias is not None:
        _refuse_bias_gradient(bias, "mxfp4_linear")
    shape = x.shape
    if len(shape) == 0 or shape[-1] != w.K:
        raise RuntimeError(f"x must be rows of {w.K}, got {tuple(shape)}")
    return _linear(x, w.codes, w.scales, w.K, bias, activation_bits)


def _expert_linear(x, codes, scales, K, rows, bias):
    if x.dim() != 2 or x.shape[1] != K or x.shape[0] * rows.k != rows.M and x.shape[0] != rows.M:
        raise RuntimeError(f"x must be [{rows.M // rows.k}, {K}] or [{rows.M}, {K}] for {rows.M} rows, got {tuple(x.shape)}")
    if codes.dim() != 3 or codes.shape[0] != rows.n:
        raise RuntimeError(f"weights of {rows.n} experts expected, got codes {tuple(codes.shape)}")
    if dm._nothing_recorded_eagerly(x):
        return ops._mx4_linear(x, codes, scales, K, bias, 16, rows.plan, rows.M)
    return _MXFP4Linear.apply(x, (codes, scales, K), bias, 16, rows)


@eager_only
def mxfp4_expert_linear(x: torch.Tensor, w: MXFP4Tensor, rows: ExpertRows, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[r] = x[r] w[e]^T + bias[e] for the expert e of every row r; w [E, N, K], bias [E, N].

    x: [T k, K], a row for every place of every token, or [T, K]: the k places of a token read its
    row, and dX is the sum over them (in fp32, rounded once).  y: [T k, N] in x's dtype, in the
    tokens' order; rows without an expert are zeros, and give no gradient.  Numerics as mxfp4_linear's."""
    _refuse_bias_gradient(bias, "mxfp4_expert_linear")
    return _expert_linear(x, w.codes, w.scales, w.K, rows, bias)


class MXFP4Linear(nn.Module):
    """A frozen linear layer whose weight is held in MXFP4, in the place of a QuantLinear (also
    inside a LoRALinear).  activation_bits=4 multiplies activations in 4 bits too."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation_bits: int = 16):
        super().__init__()
        if activation_bits not in (4, 16):
            raise ValueError(f"activation_bits must be 4 or 16, got {activation_bits}")
        self.in_features, self.out_features = in_features, out_features
        self.activation_bits = activation_bits
        pitch = ops.mx4_pad(in_features)
        # codes of zeros
        self.register_buffer("weight_quant", torch.zeros(out_features, pitch // 2, dtype=torch.uint8))
        self.register_buffer("weight_scales", torch.zeros(out_features, pitch // ops.MX4_BLOCK, dtype=torch.uint8))
        self.bias = nn.Parameter(torch.zeros(out_features), requires_grad=False) if bias else None

    @classmethod
    def from_linear(cls, linear: nn.Linear, activation_bits: int = 16) -> "MXFP4Linear":
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, activation_bits)
        t = quantize_mxfp4(linear.weight)
        m.weight_quant, m.weight_scales = t.codes, t.scales
        if linear.bias is not None:
            m.bias = nn.Parameter(linear.bias.detach().clone(), requires_grad=False)
        return m

    def dequantized_weight(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return dequantize_mxfp4(MXFP4Tensor(self.weight_quant, self.weight_scales, self.in_features), dtype)

    @eager_only
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _refuse_bias_gradient(self.bias, "MXFP4Linear")
        ops._check_mx4(self.weight_quant, self.weight_scales, self.in_features)
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise RuntimeError(f"x must be rows of {self.in_features}, got {tuple(x.shape)}")
        return _linear(x, self.weight_quant, self.weight_scales, self.in_features, self.bias, self.activation_bits)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"activation_bits={self.activation_bits}")


class MXFP4Experts(nn.Module):
    """The frozen linear layers of n experts, held in MXFP4: one grouped product for a batch whose
    rows go to experts of their own."""

    def __init__(self, n: int, in_features: int, out_features: int, bias: bool = False):
        super().__init__()
        self.n, self.in_features, self.out_features = n, in_features, out_features
        pitch = ops.mx4_pad(in_features)
        self.register_buffer("weight_quant", torch.zeros(n, out_features, pitch // 2, dtype=torch.uint8))
        self.register_buffer("weight_scales", torch.zeros(n, out_features, pitch // ops.MX4_BLOCK, dtype=torch.uint8))
        self.bias = nn.Parameter(torch.zeros(n, out_features), requires_grad=False) if bias else None

    @classmethod
    @torch.no_grad()
    def from_weights(cls, weights: Union[torch.Tensor, nn.ModuleList, list], bias: Optional[torch.Tensor] = None) -> "MXFP4Experts":
        """From stacked weights [n, out, in] (and bias [n, out]), or a list of nn.Linear layers of one
        shape, quantized one expert at a time."""
        layers = None
        if not isinstance(weights, torch.Tensor):
            layers = list(weights)
            weights = [m.weight for m in layers]
        elif weights.dim() != 3:
            raise RuntimeError(f"weights must be [experts, out, in], got {tuple(weights.shape)}")
        if len(weights) == 0:
            raise ValueError("no experts given")
        out, cols = weights[0].shape
        if any(tuple(w.shape) != (out, cols) for w in weights):
            raise ValueError("experts' weights differ in shape")
        if layers and bias is None and any(m.bias is not None for m in layers):
            if any(m.bias is None for m in layers):
                raise ValueError("all experts have a bias, or none")
            bias = torch.stack([m.bias.detach() for m in layers])
        m = cls(len(weights), cols, out, bias is not None)
        held = [quantize_mxfp4(w) for w in weights]
        m.weight_quant = torch.stack([t.codes for t in held])
        m.weight_scales = torch.stack([t.scales for t in held])
        if bias is not None:
            if tuple(bias.shape) != (m.n, out):
                raise RuntimeError(f"bias must be {(m.n, out)}, got {tuple(bias.shape)}")
            m.bias = nn.Parameter(bias.detach().clone(), requires_grad=False)
        return m

    @eager_only
    def forward(self, x: torch.Tensor, rows: ExpertRows) -> torch.Tensor:
        _refuse_bias_gradient(self.bias, "MXFP4Experts")
        ops._check_mx4(self.weight_quant, self.weight_scales, self.in_features)
        return _expert_linear(x, self.weight_quant, self.weight_scales, self.in_features, rows, self.bias)

    def extra_repr(self) -> str:
        return f"n={self.n}, in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
