"""MXFP4 and the linears on it by their definitions, in 64 bits on the CPU."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """codes (one a value), scale bytes and values (fp64) of rows [M, K], padded to whole 128 columns."""
    v = x.detach().double().cpu().numpy()
    M, K = v.shape
    pitch = -(-K // 128) * 128
    pad = np.zeros((M, pitch))
    pad[:, :K] = v
    b = pad.reshape(M, pitch // 32, 32)
    top = np.abs(b).max(2)
    fine = np.isfinite(b).all(2)
    safe = np.where(fine & (top > 0), top, 1.0)
    e = np.clip(np.frexp(safe)[1] - 1 - 2, -127, 127)
    e = np.where(top == 0, -127, e)
    a = np.where(fine[:, :, None], np.abs(b), 0.0) * np.exp2(-e.astype(np.float64))[:, :, None]
    # nearest of the grid, ties to the even code
    mid = (GRID[1:] + GRID[:-1]) / 2
    lo, hi = np.searchsorted(mid, a, side="left"), np.searchsorted(mid, a, side="right")
    mag = np.where(lo % 2 == 0, lo, hi)
    neg = np.signbit(b) & fine[:, :, None]
    codes = (mag + 8 * neg).reshape(M, pitch)
    scales = np.where(fine, e + 127, 255)
    return codes.astype(np.int64), scales.astype(np.int64), values(codes, scales)


def values(codes, scales):
    """The values (fp64) that codes (one a value, [M, Kp]) and scale bytes [M, Kp / 32] stand for."""
    M, pitch = codes.shape
    mag = GRID[codes & 7] * np.where(codes >= 8, -1.0, 1.0)
    unit = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (mag.reshape(M, -1, 32) * unit[:, :, None]).reshape(M, pitch)


def unpack(packed):
    """Packed bytes [..., n] as codes [..., 2 n]."""
    p = packed.cpu().numpy().astype(np.int64)
    return np.stack([p & 15, p >> 4], -1).reshape(*p.shape[:-1], -1)


def held(codes, scales, K):
    """The values (fp64 tensor [..., K]) of packed codes [..., Kp / 2] and scales [..., Kp / 32]."""
    c = unpack(codes.reshape(-1, codes.shape[-1]))
    v = values(c, scales.reshape(-1, scales.shape[-1]).cpu().numpy().astype(np.int64))
    return torch.from_numpy(v).reshape(*codes.shape[:-1], -1)[..., :K].contiguous()


def tolerance(dtype, y, terms, size):
    """How far a result may be from y (64 bits): half a step of its type, and for the fp32 sum of `terms`
    products, whose magnitudes add up to `size`, one step of fp32 for each addition (the rounding of
    the matrix units' additions is taken to be a whole step at most)."""
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half * 2
    acc = (terms + 2) * 2.0 ** -23 * size
    return acc + half * (y.abs() + acc) + tiny
