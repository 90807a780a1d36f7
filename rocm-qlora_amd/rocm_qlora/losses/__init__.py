"""Losses on a language model's logits (no counterpart in the reference)."""
from rocm_qlora.losses.preference import preference_loss, sequence_logps

__all__ = ["preference_loss", "sequence_logps"]
