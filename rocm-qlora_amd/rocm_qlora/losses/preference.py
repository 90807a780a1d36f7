"""Preference loss on paired log ratios, and the log-probabilities under it.

With L_i the log-probability of sequence i's labelled tokens and R_i the
reference model's,
    D_p = beta ((L_chosen - R_chosen) - (L_rejected - R_rejected))
    loss = mean over pairs of -(1 - e) log sigmoid(D_p) - e log sigmoid(-D_p),
e = label_smoothing.  One pass over the labelled rows of the logits forward,
one more backward, which writes the logits' gradient; sums over rows are fp64.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from rocm_qlora import ops
from rocm_qlora.kernels.dequant_matmul import _nothing_recorded_eagerly
from rocm_qlora.torch_ops import eager_only, first_order


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, offsets, ref_logps, beta, label_smoothing, average, ignore_index):
        loss, logps, state = ops.preference_forward(logits, labels, offsets, ref_logps, beta=beta,
                                                    label_smoothing=label_smoothing, average=average,
                                                    ignore_index=ignore_index)
        ctx.save_for_backward(logits, state)
        ctx.mark_non_differentiable(logps)
        return loss, logps

    @staticmethod
    @first_order
    def backward(ctx, dloss, _):
        logits, state = ctx.saved_tensors
        return (ops.preference_backward(logits, state, dloss),) + (None,) * 7


class _SequenceLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, offsets, average, ignore_index):
        _, logps, state = ops.preference_forward(logits, labels, offsets, average=average, ignore_index=ignore_index,
                                                 pairs=False)
        ctx.save_for_backward(logits, state)
        return logps

    @staticmethod
    @first_order
    def backward(ctx, dlogps):
        logits, state = ctx.saved_tensors
        return (ops.preference_backward(logits, state, dlogps),) + (None,) * 4


@eager_only
def preference_loss(logits: torch.Tensor, labels: torch.Tensor, offsets: Optional[torch.Tensor] = None,
                    ref_logps: Optional[torch.Tensor] = None, *, beta: float = 0.1, label_smoothing: float = 0.0,
                    average: bool = False, ignore_index: int = -100) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, logps) of P pairs of sequences, the P chosen ones first.

    logits: [T, V] packed, sequence i being rows offsets[i] to offsets[i + 1] - 1
    (offsets int32 or int64, [2 P + 1]), or [2 P, L, V] padded; fp32, bf16 or fp16.
    labels: int64, in the positions of their tokens: row t of a sequence predicts
    labels[t + 1], and positions labelled ignore_index (prompts, padding) do not
    count.  A label outside the vocabulary makes its sequence NaN.
    ref_logps: the reference model's sequence_logps, [2 P] (None: zeros).
    average: log-probabilities per labelled token instead of their sum.
    loss is differentiable by the logits; logps [2 P] (fp32) is not."""
    if _nothing_recorded_eagerly(logits):
        return ops.preference_forward(logits, labels, offsets, ref_logps, beta=beta, label_smoothing=label_smoothing,
                                      average=average, ignore_index=ignore_index)[:2]
    return _PreferenceLoss.apply(logits, labels, offsets, ref_logps, float(beta), float(label_smoothing), bool(average),
                                 int(ignore_index))


@eager_only
def sequence_logps(logits: torch.Tensor, labels: torch.Tensor, offsets: Optional[torch.Tensor] = None, *,
                   average: bool = False, ignore_index: int = -100) -> torch.Tensor:
    """Log-probabilities [S] (fp32) of the labelled tokens of S sequences, laid out as
    preference_loss takes them; differentiable by the logits.  Under torch.no_grad
    these are preference_loss's ref_logps when the reference model gives the logits."""
    if _nothing_recorded_eagerly(logits):
        return ops.preference_forward(logits, labels, offsets, average=average, ignore_index=ignore_index, pairs=False)[1]
    return _SequenceLogps.apply(logits, labels, offsets, bool(average), int(ignore_index))
