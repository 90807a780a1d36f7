"""Adapters of many requests (or of many users' training batches) beside one
shared, quantized projection (no counterpart in the reference).

Every row of a batch names its adapter, or none: y[m] = base(x[m]) + s[a]
(x[m] A[a]^T) B[a]^T.  A serving step and a training step group their rows by
adapter once (AdapterRows) and pass that to every projection.  In preference
tuning the policy's rows name their adapter and the reference model's none, so
that both run as one batch.
"""
from __future__ import annotations

import math
import warnings
from typing import Optional, Union

import torch
import torch.nn as nn

from rocm_qlora import ops
from rocm_qlora._device import on
from rocm_qlora.kernels import dequant_matmul as dm
from rocm_qlora.lora.lora_layer import LoRALinear
from rocm_qlora.quantization.quant_linear import QuantLinear
from rocm_qlora.torch_ops import eager_only, first_order


class AdapterRows:
    """The rows of a batch grouped by adapter, for every projection that the batch
    passes through.  ids: [M] (or the batch's leading shape) int32 or int64 on the
    GPU, 0 .. n - 1, or anything else for rows without an adapter; made on the
    current stream, without a host synchronization."""
    __slots__ = ("M", "n", "plan")

    def __init__(self, ids: torch.Tensor, n: int):
        self.M, self.n = ids.numel(), int(n)
        self.plan = ops.adapter_rows(ids, self.n)

    @classmethod
    def single(cls, M: int) -> "AdapterRows":
        """M rows that all belong to adapter 0 of one."""
        rows = cls.__new__(cls)
        rows.M, rows.n, rows.plan = int(M), 1, None
        return rows


def _check(x: torch.Tensor, lora_a: torch.Tensor, rows: AdapterRows, activation_bits: int) -> None:
    if activation_bits not in (8, 16):
        raise ValueError(f"activation_bits must be 8 or 16, got {activation_bits}")
    if rows.n != lora_a.shape[0] or rows.M * x.shape[-1] != x.numel():
        raise RuntimeError(f"rows of {rows.M} rows and {rows.n} adapters do not fit x {tuple(x.shape)} and "
                           f"{lora_a.shape[0]} adapters")


class _MultiLoRA(torch.autograd.Function):
    """base(x) plus the adapters' term.  base: a tensor of the rows' results, None, or
    a pair (forward, dx) of a quantized linear's functions, whose result the term is
    added to in place, and likewise in the backward pass."""

    @staticmethod
    def forward(ctx, x, lora_a, lora_b, base, scaling, rows, bits, linear):
        need = ctx.needs_input_grad
        dtype = x.dtype
        a = lora_a if lora_a.dtype == dtype else lora_a.to(dtype)
        b = lora_b if lora_b.dtype == dtype else lora_b.to(dtype)
        flat = x.dim() == 2
        x2 = x if flat else x.reshape(-1, x.shape[-1])
        out = None
        if linear is not None:
            base = out = linear[0](x2)
        elif base is not None and not flat:
            base = base.reshape(-1, b.shape[1])
        y = ops.multi_lora(x2, a, b, scaling, rows.plan, base, out, need_u=need[2])
        u = None
        if need[2]:
            y, u = y
        ctx.args = (rows.plan, linear, None if flat else x.shape, lora_a.dtype, lora_b.dtype)
        held, exps = (None, None) if not need[1] else ops.act8_quantize(x2) if bits == 8 else (x2, None)
        ctx.save_for_backward(held, exps, a if a.is_contiguous() else a.contiguous(), b if b.is_contiguous() else b.contiguous(),
                              scaling, u)
        return y if flat else y.view(*x.shape[:-1], y.shape[-1])

    @staticmethod
    @first_order
    def backward(ctx, dy):
        x, exps, a, b, scaling, u = ctx.saved_tensors
        plan, linear, shape, a_dtype, b_dtype = ctx.args
        need = ctx.needs_input_grad
        dy2 = dy if shape is None else dy.reshape(-1, dy.shape[-1])
        dx = linear[1](dy2) if linear is not None and need[0] else None
        with on(dy.device):
            dx, da, db = ops._multi_lora_grads((x, exps) if exps is not None else x, dy2, a, b, scaling, plan, u, need[0],
                                               need[1], need[2], dx, dy.device)
        if da is not None and a_dtype != da.dtype:
            da = da.to(a_dtype)
        if db is not None and b_dtype != db.dtype:
            db = db.to(b_dtype)
        return dx if shape is None or dx is None else dx.view(shape), da, db, dy if need[3] else None, None, None, None, None


@eager_only
def multi_lora(x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: Union[float, torch.Tensor],
               rows: AdapterRows, base: Optional[torch.Tensor] = None, activation_bits: int = 16) -> torch.Tensor:
    """base[m] + scaling[a] (x[m] A[a]^T) B[a]^T for the adapter a of every row m.

    x: [..., K] fp32, bf16 or fp16; lora_a [n, r, K] and lora_b [n, N, r] (rounded to
    x's dtype when they have another, and so are their gradients); scaling: fp32 [n], or one number; base: [...,
    N] in x's dtype (None: zeros).  Sums are fp32; x A^T is passed to the second
    product in 16 bits or more and the result rounded once (fp16: x A^T up to 65504; an
    infinity in lora_b, or in a gradient's x, may come out as NaN).  Differentiable by x,
    lora_a, lora_b and base (not by scaling); activation_bits=8 holds x for dA as an 8-bit checkpoint
    (rocm_qlora.checkpoint), which the gradient kernel reads as it is."""
    _check(x, lora_a, rows, activation_bits)
    # (2-D rows' base is checked with the other operands)
    if base is not None and x.dim() != 2 and (base.dtype != x.dtype or base.shape[:-1] != x.shape[:-1] or
                                              base.shape[-1] != lora_b.shape[1]):
        raise RuntimeError(f"base {tuple(base.shape)} {base.dtype} does not fit x {tuple(x.shape)} {x.dtype} and "
                           f"{lora_b.shape[1]} columns")
    if not isinstance(scaling, torch.Tensor):
        scaling = torch.full((rows.n,), float(scaling), dtype=torch.float32, device=x.device)
    elif scaling.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("multi_lora has no gradient by scaling: pass it detached")
    if dm._nothing_recorded_eagerly(x, lora_a, lora_b, base):
        dtype = x.dtype
        a = lora_a if lora_a.dtype == dtype else lora_a.to(dtype)
        b = lora_b if lora_b.dtype == dtype else lora_b.to(dtype)
        if x.dim() == 2:
            return ops.multi_lora(x, a, b, scaling, rows.plan, base)
        N = lora_b.shape[1]
        y = ops.multi_lora(x.reshape(-1, x.shape[-1]), a, b, scaling, rows.plan, None if base is None else base.reshape(-1, N))
        return y.view(*x.shape[:-1], N)
    return _MultiLoRA.apply(x, lora_a, lora_b, base, scaling, rows, activation_bits, None)


def _refuse_merged(base: QuantLinear, name: str) -> None:
    """The adapters' term goes beside the quantized weight, not one that an adapter was merged into."""
    if base.merged_mode:
        raise RuntimeError(f"{name} is merged: unmerge its adapter first")


class MultiLoRALinear(nn.Module):
    """A QuantLinear with n adapters of rank r.  lora_A [n, r, in] and lora_B [n, out,
    r] are parameters (A Kaiming-uniform, B zeros, as LoRALinear's), `scaling` [n] a
    buffer.  The rows of a batch are given to forward, or set for all layers of a
    model by set_adapter_rows.  Beside 16-bit rows the parameters of all n adapters are
    rounded to the rows' dtype at every call, and their gradients are sums in fp32 that
    are rounded to it; parameters of the rows' dtype save the conversion.  The quantized
    layer's kernels are called, not its forward: hooks on base_layer do not run."""

    def __init__(self, quant_linear: QuantLinear, n: int, r: int = 8, lora_alpha: float = 16, activation_bits: int = 16):
        if not isinstance(quant_linear, QuantLinear):
            raise TypeError(f"adapters go beside a QuantLinear, got {type(quant_linear).__name__}")
        _refuse_merged(quant_linear, "the QuantLinear")
        super().__init__()
        self.base_layer = quant_linear
        self.n, self.r = n, r
        self.activation_bits = activation_bits
        self.rows: Optional[AdapterRows] = None
        for p in quant_linear.parameters():
            p.requires_grad_(False)
        dev = quant_linear.weight_quant.device
        a = torch.empty(n, r, quant_linear.in_features)
        for i in range(n):
            nn.init.kaiming_uniform_(a[i], a=math.sqrt(5))
        self.lora_A = nn.Parameter(a.to(dev))
        self.lora_B = nn.Parameter(torch.zeros(n, quant_linear.out_features, r, device=dev))
        self.register_buffer("scaling", torch.full((n,), lora_alpha / r, device=dev))

    @torch.no_grad()
    def load_adapter(self, i: int, layer: LoRALinear) -> None:
        """Adapter i from a LoRALinear of at most this rank (the ranks it lacks are zeros)."""
        if layer.r > self.r:
            raise ValueError(f"an adapter of rank {layer.r} does not fit rank {self.r}")
        self.lora_A[i].zero_()
        self.lora_B[i].zero_()
        self.lora_A[i, :layer.r].copy_(layer.lora_A)
        self.lora_B[i, :, :layer.r].copy_(layer.lora_B)
        self.scaling[i] = layer.scaling

    def _linear(self):
        """The quantized linear and its input gradient as functions of 2-D rows."""
        base = self.base_layer
        _refuse_merged(base, "the QuantLinear")
        if base.bits == 4:
            w = base.nf4_weight()
            return (lambda x: ops.nf4_linear(x, w.packed, w.scales, w.N, w.block_size, base.bias, **w.dq_kwargs()),
                    lambda dy: ops.nf4_linear_dx(dy, w.packed, w.scales, w.K, w.block_size, **w.dq_kwargs()))
        w = base.int8_weight()
        return (lambda x: ops.int8_linear(x, w.q, w.scales, w.N, w.block_size, base.bias),
                lambda dy: ops.int8_linear_dx(dy, w.q, w.scales, w.K, w.block_size))

    @eager_only
    def forward(self, x: torch.Tensor, rows: Optional[AdapterRows] = None) -> torch.Tensor:
        rows = rows if rows is not None else self.rows
        if rows is None:
            raise RuntimeError("no adapter rows: pass them, or set them with set_adapter_rows(model, rows)")
        _check(x, self.lora_A, rows, self.activation_bits)
        linear = self._linear()
        scaling = self.scaling if self.scaling.dtype == torch.float32 else self.scaling.float()  # cast with the model
        if not dm._nothing_recorded_eagerly(x, self.lora_A, self.lora_B):
            return _MultiLoRA.apply(x, self.lora_A, self.lora_B, None, scaling, rows, self.activation_bits, linear)
        x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        y = linear[0](x2)
        ops.multi_lora(x2, self.lora_A.to(x.dtype), self.lora_B.to(x.dtype), scaling, rows.plan, y, y)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[-1])

    def extra_repr(self) -> str:
        return f"adapters={self.n}, r={self.r}, activation_bits={self.activation_bits}"


def set_adapter_rows(model: nn.Module, rows: Optional[AdapterRows]) -> int:
    """Set the batch's rows by adapter on every MultiLoRALinear; returns how many."""
    count = 0
    for m in model.modules():
        if isinstance(m, MultiLoRALinear):
            m.rows = rows
            count += 1
    return count


def attach_adapters(model: nn.Module, n: int, activation_bits: int = 16) -> nn.Module:
    """Replace every LoRALinear (quantize_model's) by a MultiLoRALinear of n adapters of
    its rank over the same quantized weight; adapter 0 is the layer's own, without its
    dropout (a warning says so).  Returns the model, or what replaces it when it is a LoRALinear itself."""
    layers = [(name, m) for name, m in model.named_modules(remove_duplicate=False) if isinstance(m, LoRALinear)]
    for name, m in layers:
        if m.merged:
            raise RuntimeError(f"{name} is merged: unmerge it first")
        if not isinstance(m.base_layer, QuantLinear):
            raise TypeError(f"{name}: adapters go beside a QuantLinear, got {type(m.base_layer).__name__}")
        _refuse_merged(m.base_layer, f"{name}'s QuantLinear")
    dropout = [name for name, m in layers if isinstance(m.lora_dropout, nn.Dropout) and m.lora_dropout.p > 0.0]
    if dropout:
        warnings.warn(f"the adapters have no dropout: that of {dropout[0] or 'the layer'}"
                      f"{f' and {len(dropout) - 1} more' if len(dropout) > 1 else ''} is left out", stacklevel=2)
    made = {}  # a layer in several places stays one
    for name, m in layers:
        if m not in made:
            made[m] = MultiLoRALinear(m.base_layer, n, m.r, m.lora_alpha, activation_bits).train(m.training)
            made[m].load_adapter(0, m)
        if m is model:
            return made[m]
        parent, _, child = name.rpartition(".")
        setattr(model.get_submodule(parent), child, made[m])
    return model
