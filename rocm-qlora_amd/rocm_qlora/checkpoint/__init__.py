"""Activation checkpoints in 8 bits: what a backward pass needs of the forward's
activations, held at half the size (no counterpart in the reference)."""
from rocm_qlora.checkpoint.act8 import Act8, compress, decompress, saved_in_8_bits

__all__ = ["Act8", "compress", "decompress", "saved_in_8_bits"]
