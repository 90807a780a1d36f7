"""8-bit activation checkpoints.

Blocks of 32 values along the last dimension share a power-of-two scale: with
E = floor(log2 max |x|), a value is held as q = round(x 2^(6-E)) in -127 .. 127
and stands for q 2^(E-6) (the OCP MX format MXINT8), at most half a step of
2^(E-6) from x (a whole one where |x| > 127 steps).  Such a value is exact in
bf16, fp16 and fp32, so matrix products read the codes as operands without
rounding again.  A block with an infinity or a NaN stands for NaN.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass

import torch

from rocm_qlora import ops
from rocm_qlora.torch_ops import eager_only


@dataclass(frozen=True)
class Act8:
    """An activation's 8-bit checkpoint: codes and exponents of its rows (ops.act8_quantize)."""
    codes: torch.Tensor
    exponents: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()


@eager_only
def compress(x: torch.Tensor) -> Act8:
    """x ([..., K], fp32/bf16/fp16, on the GPU) as its 8-bit checkpoint."""
    codes, exps = ops.act8_quantize(x.detach())
    return Act8(codes, exps, x.shape, x.dtype)


@eager_only
def decompress(c: Act8) -> torch.Tensor:
    """The values that a checkpoint stands for, in the shape and dtype it was made from."""
    return ops.act8_dequantize(c.codes, c.exponents, c.shape[-1], c.dtype).view(c.shape)


# autograd nodes that leave a parameter a parameter: viewed in whatever way, copied into another
# order or cast
_VIEWS = {"TBackward0", "TransposeBackward0", "PermuteBackward0", "ViewBackward0", "UnsafeViewBackward0", "ReshapeAliasBackward0",
          "AsStridedBackward0", "AliasBackward0", "SliceBackward0", "SelectBackward0", "DiagonalBackward0", "UnfoldBackward0",
          "SplitBackward0", "SplitWithSizesBackward0", "UnsafeSplitBackward0", "UnsafeSplitWithSizesBackward0",
          "UnbindBackward0", "ExpandBackward0", "UnsqueezeBackward0", "SqueezeBackward0", "SqueezeBackward1",
          "SqueezeBackward2", "CloneBackward0", "ToCopyBackward0"}


def _floats(t: torch.Tensor, min_elements: int) -> bool:
    return t.is_cuda and t.dtype in (torch.float32, torch.bfloat16, torch.float16) and t.dim() > 0 and \
        t.numel() >= max(min_elements, 1) and not isinstance(t, torch.nn.Parameter)


def _activation(t: torch.Tensor) -> bool:
    """Whether t was computed from more than a parameter: autograd records how, and the
    record does not lead through views, copies and casts alone to a parameter.  (What has no
    record may be a frozen weight.)"""
    node = t.grad_fn
    while node is not None and node.name() in _VIEWS:
        node = node.next_functions[0][0]
    return node is not None and node.name() != "struct torch::autograd::AccumulateGrad" and \
        node.name() != "torch::autograd::AccumulateGrad"


@contextmanager
def _saved(holds):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: compress(t) if holds(t) else t,
                                                  lambda c: decompress(c) if isinstance(c, Act8) else c):
        yield


def saved_in_8_bits(min_elements: int = 1 << 16):
    """A context in which autograd holds the float activations that it saves for the
    backward pass in 8 bits: GPU tensors of at least min_elements values that were
    computed from a tensor that requires a gradient.  Parameters, their views, copies and
    casts, and what requires no gradient stay as they are.  Gradients are then those at the held
    values; what the forward returns does not change.  For the activations of linears and
    gates; keep ops that differentiate small differences (norms, softmax) outside."""
    return _saved(lambda t: _floats(t, min_elements) and _activation(t))


def inputs_saved_in_8_bits(x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor):
    """The same for the input x of one layer with the factors lora_a [r, K] and lora_b [N,
    r] (and what dropout makes of x), whether or not it requires a gradient: inside the
    layer's own autograd function saved tensors have no record; where torch's products
    compose the layer, x shares its memory and dropout its name, and the factors and the
    first product stay as they are.  Where one of those has x's shape (a batch of r rows),
    what has neither a record nor x's memory stays as it is."""
    (r, K), N = lora_a.shape, lora_b.shape[0]
    shape, place = (x.numel(), x.shape[-1:]), x.untyped_storage().data_ptr()
    factors = {f.untyped_storage().data_ptr() for f in (lora_a, lora_b)}
    # A, B, their transposes' and casts', and x A^T
    alike = r == K or shape in ((r * K, (K,)), (N * r, (r,)), (N * r, (N,)))

    def holds(t: torch.Tensor) -> bool:
        if not _floats(t, 1) or (t.numel(), t.shape[-1:]) != shape:
            return False
        at = t.untyped_storage().data_ptr()
        if at == place or at in factors:
            return at == place
        node = t.grad_fn
        while node is not None and node.name() in _VIEWS:
            node = node.next_functions[0][0]
        return not alike if node is None else node.name() == "NativeDropoutBackward0"

    return _saved(holds)
