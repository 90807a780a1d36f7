"""Activation checkpoints in 8 bits: what a backward pass needs of the forward's
activations, held at half the size of 16 bits (no counterpart in the reference).
Each layer that saves a tensor holds codes of its own."""
from rocm_qlora.checkpoint.act8 import Act8, compress, decompress, saved_in_8_bits

__all__ = ["Act8", "compress", "decompress", "saved_in_8_bits"]
