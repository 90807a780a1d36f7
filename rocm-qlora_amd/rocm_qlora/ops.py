"""Functional entry points of the MI355X quantized-linear path.

Each function validates and lays out torch tensors, then calls one C-ABI
entry point of librocm_qlora_amd.so on the current HIP stream.  There is no
CPU or library fallback for any activation dtype or shape: a tensor off the
GPU, or a missing library, raises.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from rocm_qlora import _native as nat
from rocm_qlora._device import on

# activation rows up to which the NF4 linear runs as a weight-streaming GEMV
# (kGemvMaxM in csrc/rq_linear.h); above it, the MFMA GEMM
GEMV_MAX_M = 16
# rows up to which a 16-bit call may run on the skinny kernel (kSkRows in
# csrc/skinny_linear.hip)
SKINNY_MAX_M = 64
# largest N * (row stride of LoRA B) the decode GEMV addresses (2^29 elements)
GEMV_MAX_B_ELEMS = 1 << 29


def _rows(t: torch.Tensor, K: int) -> Tuple[torch.Tensor, int]:
    """[..., K] -> 2-D [rows, K] view with unit inner stride, and its row stride."""
    t2 = t if t.dim() == 2 and t.shape[1] == K else t.reshape(-1, K)
    rows, (ld, inner) = t2.shape[0], t2.stride()
    if inner != 1 or (rows > 1 and ld < K):
        t2 = t2.contiguous()
        ld = t2.stride(0)
    return t2, (ld if rows > 1 else K)


def _flat(t: torch.Tensor) -> torch.Tensor:
    """t as contiguous 1-D."""
    return (t if t.dim() == 1 else t.reshape(-1)).contiguous()


# rq_nf4_linear's workspace.  Its first RQ_LINEAR_SYNC_BYTES
# (include/rocm_qlora_amd.h) are a synchronization area that must be zero
# before the buffer's first call and that every call leaves ready for the
# next one once its kernels are done, so one buffer, zeroed once on the
# stream that uses it, serves every call ordered on that stream.  Calls that may run at the same time need buffers of their
# own, hence the keys:
#   * eager calls: one buffer per (device, stream), zeroed by a fill kernel
#     on that stream when it is created; it grows by reallocation (a dropped
#     buffer returns to torch's caching allocator, which hands it out again
#     only in stream order);
#   * graph capture: one buffer per (device, capture, stream) -- the branches
#     of a capture that forks side streams each get their own.  It is taken
#     from a pool of pre-zeroed buffers (_CAPTURE_POOL_ENTRIES of
#     _CAPTURE_POOL_BYTES per device, zeroed at the device's first eager
#     call; and every eager call that finds no free entry as large as its own
#     workspace adds one, zeroed, with one stream synchronization, up to
#     _CAPTURE_POOL_LIMIT bytes per device), so the graph needs no fill node:
#     it holds zeros before the first replay and every replay leaves it ready
#     for the next.  Captures are normally preceded by an eager warm-up call
#     of the same work, which leaves an entry of the size the capture needs.
#     Such a buffer is held for the life of the process (the graph may replay
#     it at any time).  A capture on a device without the pool, or finding
#     no free entry large enough, allocates one from the graph's private
#     memory pool (so it lives exactly as long as the graph), zeroed by a
#     fill kernel recorded in the graph, which every replay runs before the
#     captured calls.
LINEAR_SYNC_BYTES = 131328
_LINEAR_WS: dict = {}
_CAPTURE_WS: dict = {}
_WS_MIN_BYTES = 1 << 20
_CAPTURE_POOL_ENTRIES = 32
# 2 MiB holds the decode GEMV's largest workspace (M = 16 with its K-split
# partials) for the common layer shapes, so that a capture's calls share one
# pre-zeroed buffer rather than recording a fill kernel at each larger need
_CAPTURE_POOL_BYTES = 2 << 20
_CAPTURE_POOL_LIMIT = 1 << 30  # pre-zeroed capture buffers per device, at most (bytes)
_CAPTURE_POOL: dict = {}       # device index -> pre-zeroed buffers not yet handed out
_CAPTURE_POOL_BASE: dict = {}  # device index -> the allocations they are views of (kept for good)
_CAPTURE_POOL_TOTAL: dict = {}  # device index -> bytes of those allocations
_CAPTURE_POOL_MAX: dict = {}   # device index -> size of the largest buffer not yet handed out


def _ensure_capture_pool(dev, idx: int, need: int) -> None:
    """The device's pool exists and holds a free entry of at least `need`
    bytes (while the pool stays within _CAPTURE_POOL_LIMIT)."""
    if _CAPTURE_POOL_MAX.get(idx, -1) >= need:
        return
    if idx not in _CAPTURE_POOL_BASE:
        base = torch.zeros(_CAPTURE_POOL_ENTRIES * _CAPTURE_POOL_BYTES, dtype=torch.uint8, device=dev)
        torch.cuda.current_stream(dev).synchronize()  # zero before any later capture, on any stream, replays it
        _CAPTURE_POOL_BASE[idx] = [base]
        _CAPTURE_POOL_TOTAL[idx] = base.numel()
        _CAPTURE_POOL[idx] = [base[i * _CAPTURE_POOL_BYTES:(i + 1) * _CAPTURE_POOL_BYTES]
                              for i in range(_CAPTURE_POOL_ENTRIES)]
    pool = _CAPTURE_POOL[idx]
    _CAPTURE_POOL_MAX[idx] = max((e.numel() for e in pool), default=0)
    if _CAPTURE_POOL_MAX[idx] >= need:
        return
    size = -(-max(need, _CAPTURE_POOL_BYTES) // _CAPTURE_POOL_BYTES) * _CAPTURE_POOL_BYTES
    if _CAPTURE_POOL_TOTAL[idx] + size > _CAPTURE_POOL_LIMIT:
        return
    buf = torch.zeros(size, dtype=torch.uint8, device=dev)
    torch.cuda.current_stream(dev).synchronize()
    _CAPTURE_POOL_BASE[idx].append(buf)
    _CAPTURE_POOL_TOTAL[idx] += size
    pool.append(buf)
    _CAPTURE_POOL_MAX[idx] = size


def _zeroed_area(nbytes: int, dev, min_bytes: int = _WS_MIN_BYTES) -> torch.Tensor:
    ws = torch.empty(max(nbytes, min_bytes), dtype=torch.uint8, device=dev)
    ws[:LINEAR_SYNC_BYTES].zero_()
    return ws


def _workspace(x_dtype: torch.dtype, M: int, K: int, N: int, rank: int, dev) -> Optional[torch.Tensor]:
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    need = _bytes("rq_nf4_linear_workspace_size", idx, nat.dtype_code(x_dtype), M, K, N, rank)
    if need == 0:
        return None
    stream = nat.stream_handle(dev)
    if torch.cuda.is_current_stream_capturing():
        cid = nat.capture_id(dev)
        # the buffers of captures that have ended belong to their graphs'
        # pools and are dropped here; a capture still running (on another
        # stream or thread) keeps its buffer, since its pool could otherwise
        # hand the memory to a later allocation of the same capture
        for k in [k for k in _CAPTURE_WS if k[0] == idx and k[1] != cid]:
            if nat.stream_capture_id(k[2]) != k[1]:
                del _CAPTURE_WS[k]
        key = (idx, cid, stream)
        ws = _CAPTURE_WS.get(key)
        if ws is None or ws.numel() < need:
            # a larger buffer replaces a smaller one for the calls captured
            # from here on; calls captured before keep theirs
            pool = _CAPTURE_POOL.get(idx) or []
            fits = [i for i, e in enumerate(pool) if e.numel() >= need]
            if fits:
                ws = pool.pop(min(fits, key=lambda i: pool[i].numel()))
                _CAPTURE_POOL_MAX[idx] = max((e.numel() for e in pool), default=0)
            else:
                ws = _zeroed_area(need, dev, min_bytes=LINEAR_SYNC_BYTES)
            _CAPTURE_WS[key] = ws
        return ws
    _ensure_capture_pool(dev, idx, need)
    key = (idx, stream)
    ws = _LINEAR_WS.get(key)
    if ws is None or ws.numel() < need:
        ws = _zeroed_area(max(need, 2 * ws.numel() if ws is not None else 0), dev)
        _LINEAR_WS[key] = ws
    return ws


@functools.lru_cache(maxsize=4096)
def _bytes(size_fn: str, device_index, *args) -> int:
    """What the library's size query `size_fn` reports for sizes and dtype codes
    (a function of those and the current device's compute units alone)."""
    nbytes = ctypes.c_int64(0)
    nat.call(size_fn, *args, ctypes.byref(nbytes))
    return nbytes.value


def _step(dtype: torch.dtype) -> int:
    """Elements of one 128-byte k step of the dense GEMM's activations."""
    return 32 if dtype == torch.float32 else 64


def _scratch(size_fn: str, dev, *args) -> Optional[torch.Tensor]:
    """Scratch memory for one call, of the size `size_fn` reports (None when
    none is used): from torch's caching allocator, which hands it out again in
    stream order once the tensor is dropped."""
    n = _bytes(size_fn, dev.index, *args)
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


# Devices that had no room for a call's scratch memory: the smallest size that
# failed, the calls to go without it after the last failure, and those left.  A
# failed allocation makes torch give back its cached blocks to the driver, so on a
# GPU that stays full the tries are 1, 2, 4 .. _FULL_MOST_CALLS calls apart.
_FULL: dict = {}
_FULL_MOST_CALLS = 256


def _spare(size_fn: str, dev, *args) -> Optional[torch.Tensor]:
    """_scratch for a call that also runs without it: None on a GPU whose memory
    is too full for the decoded weight."""
    full = _FULL.get(dev.index)
    counts = full is not None and _bytes(size_fn, dev.index, *args) >= full[0]
    if counts and full[2] > 0:
        _FULL[dev.index] = (full[0], full[1], full[2] - 1)
        return None
    try:
        t = _scratch(size_fn, dev, *args)
    except torch.OutOfMemoryError:
        n, wait = _bytes(size_fn, dev.index, *args), 1
        if full is not None:
            n, wait = min(n, full[0]), min(2 * full[1], _FULL_MOST_CALLS)
        _FULL[dev.index] = (n, wait, wait)
        return None
    if counts:
        _FULL.pop(dev.index, None)
    return t


def nf4_linear(x: torch.Tensor, weight_quant: torch.Tensor, weight_scales: Optional[torch.Tensor],
               out_features: int, block_size: int = 64, bias: Optional[torch.Tensor] = None, *,
               c2: Optional[torch.Tensor] = None, c2_scales: Optional[torch.Tensor] = None,
               blocksize_2: int = 256, use_fp8_c2: bool = True,
               lora_a: Optional[torch.Tensor] = None, lora_b: Optional[torch.Tensor] = None,
               scaling: float = 0.0, lora_x: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x . dequant(W)^T + bias (+ LoRA) for an NF4 weight stored flat
    (quant_linear.py:182-197 and lora_layer.py:60-70 in one kernel launch
    sequence).  x: [..., K] bf16/fp16 (bf16/fp16 MFMA kernels) or fp32 (the
    fp32-MFMA kernel, everything in fp32 as the reference computes it) on the
    GPU; output has x's dtype.  Any K and block size: shapes the specialized
    kernels do not take (K % 64 != 0, other block sizes, fp32 with rank > 64)
    run on the library's generic kernels with the same roundings."""
    K = x.shape[-1]
    N = int(out_features)
    xcode = nat.dtype_code(x.dtype)
    dq = c2 is not None
    scales = c2_scales if dq else weight_scales
    dev = nat.require_gpu(x, weight_quant, scales, bias, lora_a, lora_b, c2)
    if weight_quant.dtype != torch.uint8:
        raise TypeError(f"NF4 weight_quant must be uint8, got {weight_quant.dtype}")
    if weight_quant.numel() * 2 < N * K:
        raise RuntimeError(f"weight_quant holds {weight_quant.numel() * 2} codes, need {N}x{K}")
    packed, scales = _flat(weight_quant), _flat(scales)
    if block_size < 1:
        raise RuntimeError(f"block_size must be positive, got {block_size}")
    n_blocks = -(-N * K // block_size)
    if dq:
        if c2.numel() < n_blocks or scales.numel() * blocksize_2 < n_blocks:
            raise RuntimeError("c2 / c2_scales too short for the weight")
    elif scales.numel() < n_blocks:
        raise RuntimeError(f"weight_scales holds {scales.numel()} values, need {n_blocks}")
    with on(dev):
        x2, ldx = _rows(x, K)
        M = x2.shape[0]
        # the decode GEMV reads any alignment; every other kernel whose rows are
        # whole 128-byte steps reads activations 16 bytes at a time
        fast_shape = K % 64 == 0 and block_size >= 64 and not block_size & (block_size - 1) and K % block_size == 0
        wide = K % _step(x.dtype) == 0 and (M > GEMV_MAX_M or x.dtype == torch.float32 or not fast_shape)
        if wide:
            x2, ldx = _aligned_rows(x2, K)
        y = torch.empty((M, N), dtype=x.dtype, device=dev)
        if M == 0:
            return y.reshape(*x.shape[:-1], N)
        rank = 0
        la = lb = xl = None
        ldxl = ldb = 0
        lcode = 0
        if lora_a is not None and lora_b is not None and lora_a.shape[0] > 0:
            rank = lora_a.shape[0]
            if lora_a.shape[1] != K or lora_b.shape != (N, rank):
                raise RuntimeError(f"LoRA shapes {tuple(lora_a.shape)} / {tuple(lora_b.shape)} do not fit "
                                   f"{N}x{K}")
            if lora_a.dtype not in (torch.float32, x.dtype):
                lora_a = lora_a.float()
            if lora_b.dtype != lora_a.dtype:
                lora_b = lora_b.to(lora_a.dtype)
            la = lora_a.contiguous()
            # B rows may be strided (a column slice of a wider parameter);
            # the decode GEMV addresses B with 32-bit offsets, so a stride
            # that would overflow them is packed first
            lb, ldb = _rows(lora_b, rank)
            if M <= GEMV_MAX_M and N * ldb > GEMV_MAX_B_ELEMS:
                lb, ldb = lb.contiguous(), rank
            lcode = nat.dtype_code(la.dtype)
            if lora_x is not None:
                xl, ldxl = (_aligned_rows if wide else _rows)(lora_x.to(x.dtype), K)
                if xl.shape[0] != M or xl.device != dev:
                    raise RuntimeError(f"lora_x has {xl.shape[0]} rows on {xl.device}, x {M} on {dev}")
        b = bias.contiguous() if bias is not None else None
        scratch = None
        if (M > GEMV_MAX_M or not fast_shape) and max(ldx, ldxl) * M * x.element_size() < 1 << 32:
            scratch = _spare("rq_nf4_linear_scratch_size", dev, xcode, M, K, N, block_size, rank)
        # a dense call needs no workspace beside its scratch memory; the skinny
        # kernel counts its splits in the workspace's synchronization area
        ws = _workspace(x.dtype, M, K, N, rank, dev) if scratch is None or (fast_shape and M <= SKINNY_MAX_M) else None
        codes = c2.reshape(-1).view(torch.uint8).contiguous() if dq else None
        nat.call("rq_nf4_linear_scratch",
                 x2.data_ptr(), xcode, M, K, ldx,
                 packed.data_ptr(), N, block_size, scales.data_ptr(), nat.dtype_code(scales.dtype),
                 nat.ptr(codes), nat.C2_FP8_E4M3FNUZ if use_fp8_c2 else nat.C2_INT8, blocksize_2,
                 nat.ptr(b), nat.dtype_code(b.dtype) if b is not None else 0,
                 nat.ptr(xl), ldxl, nat.ptr(la), nat.ptr(lb), ldb, lcode, rank, float(scaling),
                 y.data_ptr(), N, nat.ptr(ws), ws.numel() if ws is not None else 0,
                 nat.ptr(scratch), scratch.numel() if scratch is not None else 0, nat.stream_handle(dev))
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)


def _check_lora_g(lora_g: torch.Tensor, M: int, rank: int, dtype: torch.dtype) -> None:
    """Raise unless lora_g is what lora_grads returns for M rows of dtype and this
    rank: the dX kernels read [M, rank rounded up to 16] values behind its pointer."""
    if rank == 0:
        raise RuntimeError("lora_g without the adapter's factors")
    if dtype == torch.float32 or lora_g.dtype != dtype or lora_g.shape != (M, -(-rank // 16) * 16) or \
            not lora_g.is_contiguous():
        raise RuntimeError(f"lora_g {tuple(lora_g.shape)} {lora_g.dtype} (contiguous: {lora_g.is_contiguous()}) is not "
                           f"lora_grads' operand of {M} rows, rank {rank}, {dtype} (16-bit only)")


def _mask_rows(lora_mask: torch.Tensor, M: int, K: int, dev: torch.device) -> Tuple[torch.Tensor, int]:
    """The dropout mask's M rows of K bytes, and their stride."""
    mk, ldm = _rows(lora_mask.reshape(-1, K).view(torch.uint8), K)
    if mk.shape[0] != M or mk.device != dev:
        raise RuntimeError(f"lora_mask has {mk.shape[0]} rows on {mk.device}, dY {M} on {dev}")
    return mk, ldm


def nf4_linear_dx(dy: torch.Tensor, weight_quant: torch.Tensor, weight_scales: Optional[torch.Tensor],
                  in_features: int, block_size: int = 64, *,
                  c2: Optional[torch.Tensor] = None, c2_scales: Optional[torch.Tensor] = None,
                  blocksize_2: int = 256, use_fp8_c2: bool = True,
                  lora_a: Optional[torch.Tensor] = None, lora_b: Optional[torch.Tensor] = None,
                  scaling: float = 0.0, lora_mask: Optional[torch.Tensor] = None,
                  mask_scale: float = 1.0, lora_g: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dX = dY . dequant(W) (+ the LoRA term ((dY * s) . B) . A) for an NF4
    weight stored flat (dequant_matmul.py:338-351, lora_layer.py:67
    differentiated).  With lora_mask (the dropout mask of the adapter's input,
    [..., K] bool), the LoRA term goes through dropout's backward: times
    mask * mask_scale.  lora_g: the adapter's (dY * s) . B as lora_grads returns
    it (16-bit dY), when the caller has it.  dy: [..., N] fp32/bf16/fp16 on the GPU; output
    [..., K] in dy's dtype.  Shapes outside the MFMA dX kernel's (N or K not
    multiples of 64, other block sizes, fp32 dy) run on the generic kernels."""
    N = dy.shape[-1]
    K = int(in_features)
    dq = c2 is not None
    scales = c2_scales if dq else weight_scales
    dev = nat.require_gpu(dy, weight_quant, scales, lora_a, lora_b, c2, lora_g)
    if weight_quant.dtype != torch.uint8:
        raise TypeError(f"NF4 weight_quant must be uint8, got {weight_quant.dtype}")
    if weight_quant.numel() * 2 < N * K:
        raise RuntimeError(f"weight_quant holds {weight_quant.numel() * 2} codes, need {N}x{K}")
    packed, scales = _flat(weight_quant), _flat(scales)
    lead = dy.shape[:-1]
    with on(dev):
        # the dX kernels load dY rows 16 bytes at a time
        dy2, lddy = _aligned_rows(dy, N) if N % _step(dy.dtype) == 0 else _rows(dy, N)
        M = dy2.shape[0]
        dx = torch.empty((M, K), dtype=dy.dtype, device=dev)
        if M == 0:
            return dx.reshape(*lead, K)
        rank = 0
        la = lb = None
        ldb = 0
        lcode = 0
        if lora_a is not None and lora_b is not None and lora_a.shape[0] > 0:
            rank = lora_a.shape[0]
            if lora_a.shape[1] != K or lora_b.shape != (N, rank):
                raise RuntimeError(f"LoRA shapes {tuple(lora_a.shape)} / {tuple(lora_b.shape)} do not fit "
                                   f"{N}x{K}")
            if lora_a.dtype not in (torch.float32, dy.dtype):
                lora_a = lora_a.float()
            if lora_b.dtype != lora_a.dtype:
                lora_b = lora_b.to(lora_a.dtype)
            la = lora_a.contiguous()
            # B rows may be strided (a column slice of a wider parameter)
            lb, ldb = _rows(lora_b, rank)
            lcode = nat.dtype_code(la.dtype)
        mk, ldm = None, 0
        if rank > 0 and lora_mask is not None:
            mk, ldm = _mask_rows(lora_mask, M, K, dev)
        if lora_g is not None:
            _check_lora_g(lora_g, M, rank, dy.dtype)
        code = nat.dtype_code(dy.dtype)
        scratch = ws = None
        if lddy * M * dy.element_size() < 1 << 32:
            scratch = _spare("rq_nf4_linear_dx_scratch_size", dev, code, M, N, K, block_size, rank)
        if scratch is None:
            ws = _scratch("rq_nf4_linear_dx_workspace_size", dev, code, M, N, K, rank)
        codes = c2.reshape(-1).view(torch.uint8).contiguous() if dq else None
        nat.call("rq_nf4_linear_dx_scratch",
                 dy2.data_ptr(), nat.dtype_code(dy.dtype), M, N, lddy,
                 packed.data_ptr(), K, block_size, scales.data_ptr(), nat.dtype_code(scales.dtype),
                 nat.ptr(codes), nat.C2_FP8_E4M3FNUZ if use_fp8_c2 else nat.C2_INT8, blocksize_2,
                 nat.ptr(la), nat.ptr(lb), ldb, lcode, rank, float(scaling),
                 nat.ptr(mk), ldm, float(mask_scale),
                 dx.data_ptr(), K, nat.ptr(lora_g), nat.ptr(ws), ws.numel() if ws is not None else 0,
                 nat.ptr(scratch), scratch.numel() if scratch is not None else 0, nat.stream_handle(dev))
    return dx.reshape(*lead, K)


def lora_grads_supported(x: torch.Tensor, lora_a: torch.Tensor) -> bool:
    """Whether lora_grads takes activations and adapters like these."""
    return x.dtype in (torch.bfloat16, torch.float16) and lora_a.shape[0] <= 64 and x.numel() > 0


def lora_grads(x: torch.Tensor, dy: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: float,
               need_a: bool = True, need_b: bool = True, need_g: bool = False):
    """The adapters' gradients of x -> (x A^T) B^T * s (lora_layer.py:67
    differentiated, every intermediate in x's dtype): dB = (dY s)^T (x A^T) and
    dA = ((dY s) B)^T x, in the adapters' dtypes, and (dY s) B as nf4_linear_dx
    takes it.  x: [..., K] bf16/fp16, dy: [..., N].  Returns (dA, dB, g), None
    where not asked for."""
    K, N, rank = x.shape[-1], dy.shape[-1], lora_a.shape[0]
    dev = nat.require_gpu(x, dy, lora_a, lora_b)
    if lora_a.shape[1] != K or lora_b.shape != (N, rank):
        raise RuntimeError(f"LoRA shapes {tuple(lora_a.shape)} / {tuple(lora_b.shape)} do not fit {N}x{K}")
    with on(dev):
        x2, ldx = (_aligned_rows if K % 64 == 0 else _rows)(x, K)
        dy2, lddy = (_aligned_rows if N % 64 == 0 else _rows)(dy.to(x.dtype), N)
        M = x2.shape[0]
        if dy2.shape[0] != M:
            raise RuntimeError(f"dY has {dy2.shape[0]} rows, x {M}")
        a = lora_a if lora_a.dtype in (torch.float32, x.dtype) else lora_a.float()
        a = a.contiguous()
        b, ldb = _rows(lora_b.to(a.dtype), rank)
        da = torch.empty((rank, K), dtype=a.dtype, device=dev) if need_a else None
        db = torch.empty((N, rank), dtype=a.dtype, device=dev) if need_b else None
        g = torch.empty((M, -(-rank // 16) * 16), dtype=x.dtype, device=dev) if need_g else None
        code = nat.dtype_code(x.dtype)
        scratch = _scratch("rq_lora_grads_scratch_size", dev, code, M, K, N, rank)
        nat.call("rq_lora_grads", x2.data_ptr(), code, M, K, ldx, dy2.data_ptr(), N, lddy,
                 a.data_ptr(), b.data_ptr(), ldb, nat.dtype_code(a.dtype), rank, float(scaling),
                 nat.ptr(da), nat.ptr(db), nat.ptr(g), scratch.data_ptr(), scratch.numel(), nat.stream_handle(dev))
    return (da.to(lora_a.dtype) if need_a else None, db.to(lora_b.dtype) if need_b else None, g)


def _aligned_rows(t: torch.Tensor, K: int) -> Tuple[torch.Tensor, int]:
    """2-D [rows, K] view with a 16-byte aligned base and a row stride that
    keeps every row 16-byte aligned (the MFMA kernels load 16 bytes at a time)."""
    t2, ld = _rows(t, K)
    if t2.data_ptr() % 16 or (ld * t2.element_size()) % 16:
        t2 = t2.contiguous().clone()
        ld = K
    return t2, ld


def int8_linear(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, out_features: int,
                block_size: int = 0, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = x . (q * scale)^T + bias for int8 weights (quant_ops.py:55-78 then
    quant_linear.py:193-197).  q: [N, K] (or flat N*K) int8; block_size 0 ->
    one scale per output row ([N] scales, the row-absmax recipe), otherwise
    blockwise over the flat weight (QuantLinear bits=8 uses 64).
    x: [..., K] fp32/bf16/fp16 on the GPU; output has x's dtype.  Shapes and
    dtypes the int8 GEMV / MFMA GEMM do not take run on the generic kernels."""
    K = x.shape[-1]
    N = int(out_features)
    dev = nat.require_gpu(x, q, scales, bias)
    if q.dtype != torch.int8:
        raise TypeError(f"int8 weights expected, got {q.dtype}")
    qf = q.reshape(-1).contiguous()
    if qf.numel() < N * K:
        raise RuntimeError(f"q holds {qf.numel()} values, need {N}x{K}")
    sc = scales.reshape(-1).contiguous()
    need = N if block_size == 0 else -(-N * K // block_size)
    if sc.numel() < need:
        raise RuntimeError(f"scales hold {sc.numel()} values, need {need}")
    lead = x.shape[:-1]
    with on(dev):
        x2, ldx = _aligned_rows(x, K) if K % _step(x.dtype) == 0 else _rows(x, K)
        M = x2.shape[0]
        y = torch.empty((M, N), dtype=x.dtype, device=dev)
        if M == 0:
            return y.reshape(*lead, N)
        b = bias.contiguous() if bias is not None else None
        scratch = _spare("rq_int8_linear_scratch_size", dev, nat.dtype_code(x.dtype), M, K, N, block_size, 0, 0)
        nat.call("rq_int8_linear_scratch", x2.data_ptr(), nat.dtype_code(x.dtype), M, K, ldx,
                 qf.data_ptr(), N, block_size, sc.data_ptr(), nat.dtype_code(sc.dtype),
                 nat.ptr(b), nat.dtype_code(b.dtype) if b is not None else 0,
                 y.data_ptr(), N, nat.ptr(scratch), scratch.numel() if scratch is not None else 0,
                 nat.stream_handle(dev))
    return y.reshape(*lead, N)


def int8_linear_dx(dy: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, in_features: int,
                   block_size: int = 0, *, lora_a: Optional[torch.Tensor] = None,
                   lora_g: Optional[torch.Tensor] = None, lora_mask: Optional[torch.Tensor] = None,
                   mask_scale: float = 1.0) -> torch.Tensor:
    """dX = dY . (q * scale) for int8 weights (the backward of
    dequant_matmul.py:308-324: the dequantized weight rounded to dY's dtype,
    then the product), decoded inside the multiply.  q: [N, K] (or flat)
    int8, scales as for int8_linear; dy: [..., N] fp32/bf16/fp16 on the GPU;
    output [..., K] in dy's dtype.  With lora_g (lora_grads' (dY s) B, 16-bit
    dY) and lora_a, plus the adapter's g . A, through dropout's backward with
    lora_mask as in nf4_linear_dx."""
    N = dy.shape[-1]
    K = int(in_features)
    dev = nat.require_gpu(dy, q, scales, lora_a, lora_g)
    if q.dtype != torch.int8:
        raise TypeError(f"int8 weights expected, got {q.dtype}")
    if q.numel() < N * K:
        raise RuntimeError(f"q holds {q.numel()} values, need {N}x{K}")
    qf, sc = _flat(q), _flat(scales)
    need = N if block_size == 0 else -(-N * K // block_size)
    if sc.numel() < need:
        raise RuntimeError(f"scales hold {sc.numel()} values, need {need}")
    with on(dev):
        dy2, lddy = _aligned_rows(dy, N) if N % _step(dy.dtype) == 0 else _rows(dy, N)
        M = dy2.shape[0]
        dx = torch.empty((M, K), dtype=dy.dtype, device=dev)
        if M == 0:
            return dx.reshape(*dy.shape[:-1], K)
        rank, la, lcode, mk, ldm = 0, None, 0, None, 0
        if lora_g is not None:
            rank = lora_a.shape[0] if lora_a is not None else 0
            _check_lora_g(lora_g, M, rank, dy.dtype)
            if lora_a.shape[1] != K:
                raise RuntimeError(f"lora_a {tuple(lora_a.shape)} does not fit {M}x{K}")
            la = (lora_a if lora_a.dtype in (torch.float32, dy.dtype) else lora_a.float()).contiguous()
            lcode = nat.dtype_code(la.dtype)
            if lora_mask is not None:
                mk, ldm = _mask_rows(lora_mask, M, K, dev)
        scratch = _spare("rq_int8_linear_scratch_size", dev, nat.dtype_code(dy.dtype), M, K, N, block_size, 1, rank)
        if rank and (scratch is None or lddy * M * dy.element_size() >= 1 << 32):
            # past the dense kernel's 32-bit offsets: the adapter's term by torch
            t = lora_g[:, :rank] @ lora_a.to(dy.dtype)
            if lora_mask is not None:
                t = t * (lora_mask.reshape(-1, K).to(dy.dtype) * mask_scale)
            return int8_linear_dx(dy, q, scales, K, block_size) + t.reshape(*dy.shape[:-1], K)
        nat.call("rq_int8_linear_dx_scratch", dy2.data_ptr(), nat.dtype_code(dy.dtype), M, N, lddy,
                 qf.data_ptr(), K, block_size, sc.data_ptr(), nat.dtype_code(sc.dtype),
                 nat.ptr(lora_g) if rank else None, nat.ptr(la), lcode, rank, nat.ptr(mk), ldm, float(mask_scale),
                 dx.data_ptr(), K, nat.ptr(scratch), scratch.numel() if scratch is not None else 0,
                 nat.stream_handle(dev))
    return dx.reshape(*dy.shape[:-1], K)


def lora_add_supported(x: torch.Tensor, lora_a: torch.Tensor) -> bool:
    """Whether lora_add_ takes activations and adapters like these."""
    return x.dtype in (torch.bfloat16, torch.float16) and x.shape[-1] % 64 == 0 and 0 < lora_a.shape[0] <= 256 \
        and 0 < x.numel() // x.shape[-1] <= 1 << 20


def lora_add_(y: torch.Tensor, x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
              scaling: float) -> torch.Tensor:
    """y += (x A^T) B^T * s in place (lora_layer.py:67-70: every intermediate in
    x's dtype), for a contiguous y [..., N] in x's dtype; returns y."""
    K, N, rank = x.shape[-1], y.shape[-1], lora_a.shape[0]
    dev = nat.require_gpu(y, x, lora_a, lora_b)
    if lora_a.shape[1] != K or lora_b.shape != (N, rank):
        raise RuntimeError(f"LoRA shapes {tuple(lora_a.shape)} / {tuple(lora_b.shape)} do not fit {N}x{K}")
    if y.dtype != x.dtype or not y.is_contiguous() or y.numel() // N != x.numel() // K:
        raise RuntimeError(f"y must be contiguous [..., {N}] in {x.dtype} with x's rows")
    with on(dev):
        x2, ldx = _aligned_rows(x, K)
        M = x2.shape[0]
        a = (lora_a if lora_a.dtype in (torch.float32, x.dtype) else lora_a.float()).contiguous()
        b, ldb = _rows(lora_b.to(a.dtype), rank)
        ws = _scratch("rq_lora_add_workspace_size", dev, M, K, rank)
        nat.call("rq_lora_add", x2.data_ptr(), nat.dtype_code(x.dtype), M, K, ldx, a.data_ptr(), b.data_ptr(), ldb,
                 nat.dtype_code(a.dtype), rank, float(scaling), y.data_ptr(), N, N, ws.data_ptr(), ws.numel(),
                 nat.stream_handle(dev))
    return y


def fp8_quantize(t: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-tensor e4m3fnuz quantization of fp8_linear.py:33-42 on the GPU:
    returns (codes as torch.float8_e4m3fnuz [rows, cols], fp32 0-dim scale),
    scale = fp32(double(max|t|) / 240), codes = fnuz(RND(t / scale))."""
    dev = nat.require_gpu(t)
    t2 = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    rows, cols = t2.shape
    with on(dev):
        src, ld = _rows(t2, cols)
        codes = torch.empty((rows, cols), dtype=torch.uint8, device=dev)
        scale = torch.empty((), dtype=torch.float32, device=dev)
        ws = _scratch("rq_fp8_quantize_workspace_size", dev)
        nat.call("rq_fp8_quantize", src.data_ptr(), nat.dtype_code(t.dtype), rows, cols, ld,
                 codes.data_ptr(), scale.data_ptr(), ws.data_ptr(), ws.numel(), nat.stream_handle(dev))
    return codes.view(torch.float8_e4m3fnuz), scale


def fp8_to_e4m3fn(codes: torch.Tensor) -> torch.Tensor:
    """e4m3fnuz codes (fp8_quantize's) -> e4m3fn codes of the same values,
    the format gfx950's fp8 matrix cores read: exact except the 8 odd-mantissa
    magnitudes below 2^-6, which round to the nearest even e4m3fn code (as
    torch's .to(torch.float8_e4m3fn) does); NaN stays NaN."""
    dev = nat.require_gpu(codes)
    src = codes.view(torch.uint8).contiguous()
    with on(dev):
        out = torch.empty(src.shape, dtype=torch.uint8, device=dev)
        nat.call("rq_fp8_fnuz_to_e4m3fn", src.data_ptr(), src.numel(), out.data_ptr(), nat.stream_handle(dev))
    return out.view(torch.float8_e4m3fn)


def fp8_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """_FP8LinearFunc.forward (fp8_linear.py:27-60) for a weight quantized by
    fp8_quantize: x is quantized per tensor, the fp8 products are summed by
    the fp8 matrix cores in fp32, scaled by x_scale * w_scale, rounded to x's
    dtype, and the bias is added.  w_codes: torch.float8_e4m3fn (fp8_to_e4m3fn
    of the quantized weight, used as is) or torch.float8_e4m3fnuz / uint8
    (re-encoded on every call).  x: [..., K] fp32/bf16/fp16 on the GPU (fp32
    x, K % 64 != 0 or unaligned rows: the generic kernels, which decode the
    codes and sum the fp32 products as fp8_linear.py:44-52 does)."""
    K = x.shape[-1]
    dev = nat.require_gpu(x, w_codes, w_scale, bias)
    if w_codes.dtype != torch.float8_e4m3fn:
        if w_codes.dtype not in (torch.float8_e4m3fnuz, torch.uint8):
            raise TypeError(f"fp8 weight codes expected, got {w_codes.dtype}")
        w_codes = fp8_to_e4m3fn(w_codes)
    wc = w_codes.reshape(-1, K).view(torch.uint8).contiguous()
    N = wc.shape[0]
    ws_scale = w_scale.reshape(()).to(torch.float32).contiguous()
    lead = x.shape[:-1]
    with on(dev):
        x2, ldx = _aligned_rows(x, K) if K % 64 == 0 and x.dtype != torch.float32 else _rows(x, K)
        M = x2.shape[0]
        y = torch.empty((M, N), dtype=x.dtype, device=dev)
        if M == 0:
            return y.reshape(*lead, N)
        ws = _scratch("rq_fp8_linear_workspace_size", dev, M, K)
        b = bias.to(x.dtype).contiguous() if bias is not None else None
        nat.call("rq_fp8_linear", x2.data_ptr(), nat.dtype_code(x.dtype), M, K, ldx,
                 wc.data_ptr(), N, ws_scale.data_ptr(), nat.ptr(b),
                 nat.dtype_code(b.dtype) if b is not None else 0,
                 y.data_ptr(), N, ws.data_ptr(), ws.numel(), nat.stream_handle(dev))
    return y.reshape(*lead, N)


def int8_quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-row int8 quantization of 16-bit activations on the GPU: the
    per-row recipe of quantize_int8 (quant_ops.py:29-35) in fp32.  Returns
    (codes int8 [rows, K], scales fp32 [rows]) with scales[m] =
    max(max|x[m]| / 127, 1e-12) and codes = RNE(x / scales[m])."""
    K = x.shape[-1]
    dev = nat.require_gpu(x)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"bf16/fp16 activations expected, got {x.dtype}")
    with on(dev):
        x2, ldx = _aligned_rows(x, K)
        M = x2.shape[0]
        codes = torch.empty((M, K), dtype=torch.int8, device=dev)
        scales = torch.empty((M,), dtype=torch.float32, device=dev)
        if M:
            nat.call("rq_int8_quantize_rows", x2.data_ptr(), nat.dtype_code(x.dtype), M, K, ldx,
                     codes.data_ptr(), scales.data_ptr(), nat.stream_handle(dev))
    return codes, scales


def int8_linear_w8a8(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor,
                     bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """W8A8 INT8 mode: x quantized per row to int8 (int8_quantize_rows), the
    int8 products summed exactly in int32 by the int8 matrix cores, then
    y = RND(RND(float(acc) * x_scale[m] * w_scale[n]) + RND(bias)).
    q: [N, K] int8 with one scale per row (quantize_int8(w,
    per_channel=True)); x: [..., K] bf16/fp16 on the GPU, K % 64 == 0.
    Not the reference's INT8 linear (int8_linear: 16-bit activations times
    dequantized weights): a separate, faster mode with activation rounding."""
    K = x.shape[-1]
    dev = nat.require_gpu(x, q, scales, bias)
    if q.dtype != torch.int8:
        raise TypeError(f"int8 weights expected, got {q.dtype}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"bf16/fp16 activations expected, got {x.dtype}")
    wq = q.reshape(-1, K).contiguous()
    N = wq.shape[0]
    sc = scales.reshape(-1).contiguous()
    if sc.numel() != N:
        raise RuntimeError(f"W8A8 needs one weight scale per row: {sc.numel()} scales for {N} rows")
    lead = x.shape[:-1]
    with on(dev):
        x2, ldx = _aligned_rows(x, K)
        M = x2.shape[0]
        y = torch.empty((M, N), dtype=x.dtype, device=dev)
        if M == 0:
            return y.reshape(*lead, N)
        ws = _scratch("rq_int8_linear_w8a8_workspace_size", dev, M, K)
        b = bias.to(x.dtype).contiguous() if bias is not None else None
        nat.call("rq_int8_linear_w8a8", x2.data_ptr(), nat.dtype_code(x.dtype), M, K, ldx,
                 wq.data_ptr(), N, sc.data_ptr(), nat.dtype_code(sc.dtype), nat.ptr(b),
                 nat.dtype_code(b.dtype) if b is not None else 0,
                 y.data_ptr(), N, ws.data_ptr(), ws.numel(), nat.stream_handle(dev))
    return y.reshape(*lead, N)


MERGE_MODES = {"sum_then_round": nat.MERGE_SUM_THEN_ROUND, "round_then_sum": nat.MERGE_ROUND_THEN_SUM}


def merge_lora(weight_quant: torch.Tensor, weight_scales: torch.Tensor, out_features: int, in_features: int,
               block_size: int = 64, lora_a: Optional[torch.Tensor] = None, lora_b: Optional[torch.Tensor] = None,
               scaling: float = 0.0, *, bits: int = 4, c2: Optional[torch.Tensor] = None,
               use_fp8_c2: bool = True, blocksize_2: int = 256, mode: str = "sum_then_round",
               out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """[out, in] 16-bit weight of dequant(W) + (B @ A) * scaling, straight
    from the quantized buffers in one kernel.  mode "sum_then_round":
    RND(W + d) as LoRALinear.merge_lora rounds it (lora_layer.py:84-103);
    "round_then_sum": RND(RND(W) + RND(d)) as the export path does
    (export/gguf_export.py:53-77).  bits 4: NF4 codes with per-block absmax,
    or c2 codes with weight_scales = c2_scales under double quantization;
    bits 8: int8 codes, block_size 0 meaning one scale per row."""
    N, K = int(out_features), int(in_features)
    dev = nat.require_gpu(weight_quant, weight_scales, lora_a, lora_b, c2)
    if mode not in MERGE_MODES:
        raise ValueError(f"mode must be one of {sorted(MERGE_MODES)}, got {mode!r}")
    if out_dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"out_dtype must be float16 or bfloat16, got {out_dtype}")
    w = weight_quant.reshape(-1).contiguous()
    if bits == 4:
        fmt = nat.WEIGHT_NF4
        if w.dtype != torch.uint8 or w.numel() * 2 < N * K:
            raise RuntimeError(f"NF4 weight_quant must hold {N}x{K} codes as uint8")
    elif bits == 8:
        fmt = nat.WEIGHT_INT8
        if w.dtype != torch.int8 or w.numel() < N * K:
            raise RuntimeError(f"INT8 weight_quant must hold {N}x{K} int8 values")
    else:
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    sc = weight_scales.reshape(-1).contiguous()
    rank = 0
    la = lb = None
    ldb = lcode = 0
    if lora_a is not None and lora_b is not None and lora_a.shape[0] > 0:
        rank = lora_a.shape[0]
        if lora_a.shape[1] != K or lora_b.shape != (N, rank):
            raise RuntimeError(f"LoRA shapes {tuple(lora_a.shape)} / {tuple(lora_b.shape)} do not fit {N}x{K}")
        if lora_b.dtype != lora_a.dtype:
            lora_b = lora_b.to(lora_a.dtype)
        la = lora_a.detach().contiguous()
        lb, ldb = _rows(lora_b.detach(), rank)
        lcode = nat.dtype_code(la.dtype)
    codes = c2.reshape(-1).view(torch.uint8).contiguous() if c2 is not None else None
    with on(dev):
        out = torch.empty((N, K), dtype=out_dtype, device=dev)
        nat.call("rq_merge_lora", w.data_ptr(), fmt, N, K, block_size, sc.data_ptr(), nat.dtype_code(sc.dtype),
                 nat.ptr(codes), nat.C2_FP8_E4M3FNUZ if use_fp8_c2 else nat.C2_INT8, blocksize_2,
                 nat.ptr(la), nat.ptr(lb), ldb, lcode, rank, float(scaling), MERGE_MODES[mode],
                 out.data_ptr(), nat.dtype_code(out_dtype), K, nat.stream_handle(dev))
    return out


# ---- adapters of many requests, 8-bit activation checkpoints, preference loss -----------
ACT8_BLOCK = 32     # values that share a checkpoint's scale (kAct8Block in csrc/rq_act8.h)
MAX_ADAPTERS = 1024  # kMaxAdapters in csrc/rq_rows.h


def adapter_rows(ids: torch.Tensor, n: int) -> torch.Tensor:
    """The rows of a batch grouped by adapter: ids [M] int32 or int64 on the GPU, 0 ..
    n - 1 or, for a row without an adapter, anything else.  The result is what
    multi_lora and, for experts, mx4_linear take as `plan`, for M rows and n adapters alone: it
    carries both numbers, which a copy of its bytes (clone, to) does not."""
    dev = nat.require_gpu(ids)
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"adapter ids must be int32 or int64, got {ids.dtype}")
    if not 1 <= n <= MAX_ADAPTERS:
        raise RuntimeError(f"{n} adapters: 1 to {MAX_ADAPTERS} are taken at once")
    M = ids.numel()
    with on(dev):
        if ids.dtype == torch.int64:
            ids = ids.clamp(-1, n).to(torch.int32)  # whatever int32 cannot hold has no adapter either
        ids = ids.contiguous()
        plan = _scratch("rq_adapter_rows_size", dev, M, n)
        nat.call("rq_adapter_rows", ids.data_ptr(), M, n, plan.data_ptr(), plan.numel(), nat.stream_handle(dev))
    plan.grouped = (M, n)  # what it holds rows for: plans of other batches can have its size
    return plan


def _adapter_operands(dtype, K: int, lora_a, lora_b, scaling) -> Tuple[int, int, int, torch.Tensor, torch.Tensor]:
    """n, rank and N of stacked factors, and the factors as the kernels take them."""
    of_a, of_b = lora_a.shape, lora_b.shape
    if len(of_a) != 3 or len(of_b) != 3:
        raise RuntimeError(f"stacked factors are [n, rank, K] and [n, N, rank], got {tuple(of_a)} and {tuple(of_b)}")
    n, rank, cols = of_a
    n_b, N, rank_b = of_b
    if cols != K or n_b != n or rank_b != rank or rank < 1 or N < 1:
        raise RuntimeError(f"LoRA shapes {tuple(of_a)} / {tuple(of_b)} do not fit rows of {K}")
    if lora_a.dtype != dtype or lora_b.dtype != dtype:
        raise TypeError(f"stacked factors must have the rows' dtype {dtype}, got {lora_a.dtype} and {lora_b.dtype}")
    if scaling.dtype != torch.float32 or scaling.shape != (n,) or not scaling.is_contiguous():
        raise RuntimeError(f"scaling must be {n} contiguous fp32 values, got {tuple(scaling.shape)} {scaling.dtype}")
    return n, rank, N, lora_a.contiguous(), lora_b.contiguous()


def _check_rows(t: torch.Tensor, M: int, cols: int, dtype: torch.dtype, name: str) -> int:
    """The row stride of t, which has to be [M, cols] of dtype with adjacent columns."""
    if t.dtype == dtype and t.shape == (M, cols):
        ld, inner = t.stride()
        if M <= 1:
            ld = cols
        if ld >= cols and (inner == 1 or cols == 1):
            return ld
    raise RuntimeError(f"{name} must be [{M}, {cols}] {dtype} with adjacent columns, got {tuple(t.shape)} {t.dtype} "
                       f"of strides {t.stride()}")


def _check_plan(plan: Optional[torch.Tensor], M: int, n: int) -> None:
    """Refuses a plan of other rows, whose entries would lie outside the operands (its size can be the same)."""
    if plan is None:
        if n != 1:
            raise RuntimeError(f"{n} adapters without the batch's rows by adapter")
    elif getattr(plan, "grouped", None) != (M, n):
        raise RuntimeError(f"the rows by adapter are not those of {M} rows and {n} adapters, as adapter_rows returned them")


def multi_lora(x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: torch.Tensor,
               plan: Optional[torch.Tensor] = None, base: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, need_u: bool = False):
    """out[m] = base[m] + scaling[a] (x[m] A[a]^T) B[a]^T, a the adapter of row m in
    `plan` (None: adapter 0 of one).  x [M, K], lora_a [n, rank, K], lora_b [n, N,
    rank], base and out [M, N] (out may be base) of one dtype, scaling [n] fp32.
    Returns out and, with need_u, what multi_lora_grads takes as u."""
    dev = nat.require_gpu(x, lora_a, lora_b, scaling, plan, base, out)
    M, K = x.shape
    dtype = x.dtype
    code = nat.dtype_code(dtype)
    n, rank, N, a, b = _adapter_operands(dtype, K, lora_a, lora_b, scaling)
    ld_out = N if out is None else _check_rows(out, M, N, dtype, "out")
    ld_base = 0
    if base is not None:
        if base is out:
            ld_base = ld_out
        elif base.dtype != dtype or base.shape != (M, N):
            raise RuntimeError(f"base must be [{M}, {N}] {dtype}, got {tuple(base.shape)} {base.dtype}")
        else:
            base, ld_base = _rows(base, N)
    with on(dev):
        _check_plan(plan, M, n)
        grouped = 0 if plan is None else 1
        if out is None:
            out = x.new_empty((M, N))
        u = None
        if need_u:
            u = torch.empty(_bytes("rq_multi_lora_u_size", dev.index, M, n, rank, grouped), dtype=torch.uint8, device=dev)
        if M > 0:
            x, ldx = _rows(x, K)
            scratch = _scratch("rq_multi_lora_scratch_size", dev, code, M, K, N, n, rank, grouped, 0)
            nat.call("rq_multi_lora", x.data_ptr(), code, M, K, ldx, nat.ptr(plan), plan.numel() if grouped else 0,
                     a.data_ptr(), b.data_ptr(), scaling.data_ptr(), n, rank, N,
                     nat.ptr(base), ld_base, out.data_ptr(), ld_out, nat.ptr(u),
                     scratch.data_ptr(), scratch.numel(), nat.stream_handle(dev))
    return (out, u) if need_u else out


def multi_lora_grads(x, dy: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: torch.Tensor,
                     plan: Optional[torch.Tensor] = None, u: Optional[torch.Tensor] = None, *, need_x: bool = True,
                     need_a: bool = True, need_b: bool = True, dx: Optional[torch.Tensor] = None):
    """Gradients of multi_lora: (dx, dA, dB), None where not asked for.  x: the rows
    [M, K] or act8_quantize's (codes, exponents) of them, read for dA alone; u:
    multi_lora's, read for dB alone.  dx: [M, K], to which the adapters' input
    gradient is added (None: a new tensor of that term)."""
    dev = nat.require_gpu(dy, lora_a, lora_b, scaling, plan, u, dx)
    M, N = dy.shape
    K = lora_a.shape[-1]
    nat.dtype_code(dy.dtype)
    n, rank, n_out, a, b = _adapter_operands(dy.dtype, K, lora_a, lora_b, scaling)
    if n_out != N:
        raise RuntimeError(f"dY has {N} columns, the factors {n_out}")
    if need_a:
        if isinstance(x, tuple):
            codes, exps = x
            nat.require_gpu(dy, codes, exps)
            pitch = -(-K // ACT8_BLOCK) * ACT8_BLOCK
            if codes.shape != (M, pitch) or exps.shape != (M, pitch // ACT8_BLOCK) or codes.dtype != torch.uint8 or \
                    exps.dtype != torch.uint8 or not codes.is_contiguous() or not exps.is_contiguous():
                raise RuntimeError(f"codes {tuple(codes.shape)} / {tuple(exps.shape)} are not act8_quantize's of {M} rows of {K}")
        else:
            nat.require_gpu(dy, x)
            if x.dtype != dy.dtype or x.shape != (M, K):
                raise RuntimeError(f"x must be [{M}, {K}] {dy.dtype}, got {tuple(x.shape)} {x.dtype}")
    if dx is not None:
        _check_rows(dx, M, K, dy.dtype, "dx")
    with on(dev):
        _check_plan(plan, M, n)
        if need_b and (u is None or u.dtype != torch.uint8 or not u.is_contiguous() or
                       u.numel() != _bytes("rq_multi_lora_u_size", dev.index, M, n, rank, 0 if plan is None else 1)):
            raise RuntimeError("u is not multi_lora's of these rows and factors")
        return _multi_lora_grads(x, dy, a, b, scaling, plan, u, need_x or dx is not None, need_a, need_b, dx, dev)


def _multi_lora_grads(x, dy, a, b, scaling, plan, u, need_x, need_a, need_b, dx, dev):
    """multi_lora_grads of operands that are known to fit, on the current device."""
    M, N = dy.shape
    n, rank, K = a.shape
    base, lddx = dx, K if dx is None or M <= 1 else dx.stride(0)
    da = torch.empty_like(a) if need_a else None
    db = torch.empty_like(b) if need_b else None
    if need_x and dx is None:
        dx = dy.new_empty((M, K))
    if M == 0:
        for t in (da, db):
            if t is not None:
                t.zero_()
        return dx, da, db
    xp = exps = None
    ldx = 0
    if need_a:
        if isinstance(x, tuple):
            x, exps = x
            ldx = x.shape[1]
        else:
            x, ldx = _rows(x, K)
        xp = x.data_ptr()
    dy, lddy = _rows(dy, N)
    code = nat.dtype_code(dy.dtype)
    grouped = 0 if plan is None else 1
    scratch = _scratch("rq_multi_lora_scratch_size", dev, code, M, K, N, n, rank, grouped, 1)
    nat.call("rq_multi_lora_grads", xp, nat.ptr(exps), code, M, K, ldx, dy.data_ptr(), N, lddy,
             nat.ptr(plan), plan.numel() if grouped else 0, a.data_ptr(), b.data_ptr(), scaling.data_ptr(), n, rank,
             nat.ptr(u) if need_b else None, nat.ptr(base), lddx, nat.ptr(dx), lddx, nat.ptr(da), nat.ptr(db),
             scratch.data_ptr(), scratch.numel(), nat.stream_handle(dev))
    return dx, da, db


def act8_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The 8-bit checkpoint of x's rows ([..., K] fp32/bf16/fp16): codes [M, K rounded
    up to 32] and exponents [M, K / 32 rounded up], both uint8."""
    dev = nat.require_gpu(x)
    code = nat.dtype_code(x.dtype)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"rows expected, got shape {tuple(x.shape)}")
    K = x.shape[-1]
    with on(dev):
        x2, ldx = _rows(x, K)
        M = x2.shape[0]
        blocks = -(-K // ACT8_BLOCK)
        codes = torch.empty((M, blocks * ACT8_BLOCK), dtype=torch.uint8, device=dev)
        exps = torch.empty((M, blocks), dtype=torch.uint8, device=dev)
        nat.call("rq_act8_quantize", x2.data_ptr(), code, M, K, ldx, codes.data_ptr(), exps.data_ptr(), nat.stream_handle(dev))
    return codes, exps


def act8_dequantize(codes: torch.Tensor, exps: torch.Tensor, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """The values [M, cols] that act8_quantize's codes stand for."""
    dev = nat.require_gpu(codes, exps)
    code = nat.dtype_code(dtype)
    blocks = -(-cols // ACT8_BLOCK)
    if cols < 1 or codes.dim() != 2 or codes.shape[1] != blocks * ACT8_BLOCK or exps.shape != (codes.shape[0], blocks) or \
            codes.dtype != torch.uint8 or exps.dtype != torch.uint8:
        raise RuntimeError(f"codes {tuple(codes.shape)} / {tuple(exps.shape)} are not act8_quantize's of rows of {cols}")
    codes, exps = codes.contiguous(), exps.contiguous()
    with on(dev):
        out = torch.empty((codes.shape[0], cols), dtype=dtype, device=dev)
        nat.call("rq_act8_dequantize", codes.data_ptr(), exps.data_ptr(), codes.shape[0], cols, out.data_ptr(), code, cols,
                 nat.stream_handle(dev))
    return out


def _logit_rows(logits: torch.Tensor) -> Tuple[torch.Tensor, int, int, int, int]:
    """Logits [T, V] or [B, L, V] without a copy where the vocabulary's stride is 1:
    (tensor, T, row stride, rows a period, period stride)."""
    V = logits.shape[-1]
    if logits.stride(-1) != 1 and V > 1:
        logits = logits.contiguous()
    if logits.dim() == 2:
        T, ld = logits.shape[0], logits.stride(0)
        if T <= 1:
            return logits, T, V, 0, 0
        return (logits, T, ld, 0, 0) if ld >= V else (logits.contiguous(), T, V, 0, 0)
    B, L = logits.shape[:2]
    if (L > 1 and logits.stride(1) < V) or (B > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    ld = logits.stride(1) if L > 1 else V
    if B == 1 or logits.stride(0) == L * ld:
        return logits, B * L, ld, 0, 0
    return logits, B * L, ld, L, logits.stride(0)


def preference_forward(logits: torch.Tensor, labels: torch.Tensor, offsets: Optional[torch.Tensor] = None,
                       ref_logps: Optional[torch.Tensor] = None, *, beta: float = 0.1, label_smoothing: float = 0.0,
                       average: bool = False, ignore_index: int = -100, pairs: bool = True):
    """Log-probabilities of labelled sequences and (with `pairs`) the preference loss of
    their pairs.  logits [T, V] with offsets [S + 1] (int32/int64), or [B, L, V]: a
    sequence per batch entry; labels int64 of the logits' leading shape, in the
    positions of their tokens (row t predicts labels[t + 1]).  Returns (loss or None,
    logps [S], what preference_backward takes)."""
    dev = nat.require_gpu(logits, labels, offsets, ref_logps)
    code = nat.dtype_code(logits.dtype)
    shape = logits.shape
    dims = len(shape)
    if dims not in (2, 3) or logits.numel() == 0:
        raise RuntimeError(f"logits must be [T, V] or [B, L, V] with a row at least, got {tuple(shape)}")
    if labels.dtype != torch.int64 or labels.shape != shape[:-1]:
        raise RuntimeError(f"labels must be int64 {tuple(shape[:-1])}, got {labels.dtype} {tuple(labels.shape)}")
    if dims == 2:
        if offsets is None:
            raise RuntimeError("packed logits need their sequences' offsets")
        if offsets.dim() != 1 or offsets.numel() < 2 or offsets.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"offsets must be int32 or int64 [sequences + 1], got {offsets.dtype} {tuple(offsets.shape)}")
        S = offsets.numel() - 1
    else:
        if offsets is not None:
            raise RuntimeError("offsets go with packed logits [T, V]")
        S = shape[0]
    if pairs and S % 2:
        raise RuntimeError(f"{S} sequences are no pairs")
    if pairs and not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")
    if ref_logps is not None:
        if ref_logps.shape != (S,):
            raise RuntimeError(f"ref_logps must hold {S} values, got {tuple(ref_logps.shape)}")
        if ref_logps.dtype != torch.float32 or not ref_logps.is_contiguous():
            ref_logps = ref_logps.detach().to(torch.float32).contiguous()
    labels = labels.contiguous()
    with on(dev):
        if offsets is not None and (offsets.dtype != torch.int32 or not offsets.is_contiguous()):
            offsets = offsets.to(torch.int32).contiguous()
        z, T, ld, period, outer = _logit_rows(logits)
        V = z.shape[-1]
        # one allocation for what the backward pass keeps: 16 bytes a row, one value a sequence
        state = torch.empty(4 * T + S, dtype=torch.float32, device=dev)
        logps = torch.empty(S, dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev) if pairs else None
        ws = _scratch("rq_preference_workspace_size", dev, code, T, V, S)
        info = state.data_ptr()
        nat.call("rq_preference_forward", z.data_ptr(), code, T, V, ld, period, outer, labels.data_ptr(), nat.ptr(offsets), S,
                 int(ignore_index), nat.ptr(ref_logps), float(beta), float(label_smoothing), int(average), logps.data_ptr(),
                 nat.ptr(loss), info + 16 * T, info, ws.data_ptr(), ws.numel(), nat.stream_handle(dev))
    return loss, logps, state


def preference_backward(logits: torch.Tensor, state, grad: Optional[torch.Tensor]) -> torch.Tensor:
    """The logits' gradient, contiguous, from preference_forward's state and the
    gradient of its loss (a scalar) or of its log-probabilities ([S])."""
    dev = nat.require_gpu(logits, state, grad)
    with on(dev):
        z, T, ld, period, outer = _logit_rows(logits)
        V = z.shape[-1]
        S = state.numel() - 4 * T
        if S < 1 or state.dtype != torch.float32 or not state.is_contiguous():
            raise RuntimeError(f"state is not preference_forward's of {T} rows")
        if grad is not None:
            if grad.dtype != torch.float32 or grad.shape not in ((), (S,)):
                raise RuntimeError(f"grad must be fp32, one value or {S}, got {grad.dtype} {tuple(grad.shape)}")
            grad = grad.contiguous()
        dz = torch.empty(z.shape, dtype=z.dtype, device=dev)
        info = state.data_ptr()
        nat.call("rq_preference_backward", z.data_ptr(), nat.dtype_code(z.dtype), T, V, ld, period, outer, info, info + 16 * T,
                 nat.ptr(grad), int(grad is not None and grad.dim() > 0), dz.data_ptr(), V, nat.stream_handle(dev))
    return dz


# ---- MXFP4 weights: codec, linears, experts' linears -------------------------------------
MX4_BLOCK = 32    # values that share a scale (kMxBlock in csrc/rq_mx4.h)
MX4_WHOLE = 128   # values that a row is held in multiples of (kMxWhole)


def mx4_pad(K: int) -> int:
    """Values that a row of K is held in."""
    return -(-K // MX4_WHOLE) * MX4_WHOLE


def mx4_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The MXFP4 codes [..., Kp / 2] and scales [..., Kp / 32] (uint8; Kp = K rounded up to 128)
    of x's rows ([..., K] fp32/bf16/fp16)."""
    dev = nat.require_gpu(x)
    code = nat.dtype_code(x.dtype)
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise RuntimeError(f"rows expected, got shape {tuple(shape)}")
    K = shape[-1]
    with on(dev):
        x2, ldx = _rows(x, K)
        M = x2.shape[0]
        pitch = mx4_pad(K)
        codes = torch.empty((*shape[:-1], pitch // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((*shape[:-1], pitch // MX4_BLOCK), dtype=torch.uint8, device=dev)
        nat.call("rq_mx4_quantize", x2.data_ptr(), code, M, K, ldx, codes.data_ptr(), scales.data_ptr(), nat.stream_handle(dev))
    return codes, scales


def _check_mx4(codes: torch.Tensor, scales: torch.Tensor, K: int) -> None:
    pitch = mx4_pad(K)
    if K < 1 or codes.dim() < 1 or codes.shape[-1] * 2 != pitch or scales.shape[-1:] != (pitch // MX4_BLOCK,) or \
            codes.shape[:-1] != scales.shape[:-1]:
        raise RuntimeError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not MXFP4 rows of {K} values: "
                           f"{pitch // 2} and {pitch // MX4_BLOCK} bytes a row expected")
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"MXFP4 codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise RuntimeError("MXFP4 codes and scales must be contiguous")


def mx4_dequantize(codes: torch.Tensor, scales: torch.Tensor, K: int, dtype: torch.dtype) -> torch.Tensor:
    """The values [..., K] that mx4_quantize's codes stand for."""
    _check_mx4(codes, scales, K)
    return _mx4_dequantize(codes, scales, K, dtype)


def _mx4_dequantize(codes, scales, K, dtype):
    """mx4_dequantize of codes and scales that fit."""
    dev = nat.require_gpu(codes, scales)
    code = nat.dtype_code(dtype)
    with on(dev):
        out = torch.empty((*codes.shape[:-1], K), dtype=dtype, device=dev)
        rows = out.numel() // K
        nat.call("rq_mx4_dequantize", codes.data_ptr(), scales.data_ptr(), rows, K, out.data_ptr(), code, K,
                 nat.stream_handle(dev))
    return out


def _mx4_weight(codes: torch.Tensor, plan: Optional[torch.Tensor]) -> Tuple[int, int]:
    """Experts and rows of a weight: [N, Kp / 2] without a plan, [E, N, Kp / 2] with one."""
    shape = codes.shape
    if plan is None:
        if len(shape) != 2:
            raise RuntimeError(f"a weight's codes are [N, Kp / 2], got {tuple(shape)}")
        return 1, shape[0]
    if len(shape) != 3:
        raise RuntimeError(f"experts' codes are [E, N, Kp / 2], got {tuple(shape)}")
    return shape[0], shape[1]


def _mx4_plan(plan: torch.Tensor, M: int, E: int) -> None:
    """Refuses a plan of other rows, whose entries would lie outside the operands."""
    if getattr(plan, "grouped", None) != (M, E):
        raise RuntimeError(f"the rows by expert are not those of {M} rows and {E} experts, as adapter_rows returned them")


def _mx4_bias(bias: Optional[torch.Tensor], dtype: torch.dtype, E: int, N: int, grouped: bool) -> Optional[torch.Tensor]:
    if bias is None:
        return None
    if bias.shape != ((E, N) if grouped else (N,)):
        raise RuntimeError(f"bias must be {(E, N) if grouped else (N,)}, got {tuple(bias.shape)}")
    return bias if bias.dtype == dtype and bias.is_contiguous() else bias.detach().to(dtype).contiguous()


def mx4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, K: int, bias: Optional[torch.Tensor] = None, *,
               activation_bits: int = 16, plan: Optional[torch.Tensor] = None, M: Optional[int] = None) -> torch.Tensor:
    """y[r] = x[r / shared] W[e]^T + bias[e] on MXFP4 weights.  x: rows [R, K] fp32/bf16/fp16.
    Without a plan codes are [N, Kp / 2] and y is [R, N]; with one (adapter_rows of M rows and E
    experts) codes are [E, N, Kp / 2], y is [M, N], and M / R rows of it read one row of x."""
    _check_mx4(codes, scales, K)
    return _mx4_linear(x, codes, scales, K, bias, activation_bits, plan, M)


def _mx4_linear(x, codes, scales, K, bias, activation_bits, plan, M):
    """mx4_linear on codes and scales that fit."""
    dev = nat.require_gpu(x, codes, scales, bias, plan)
    dtype, shape = x.dtype, x.shape
    code = nat.dtype_code(dtype)
    E, N = _mx4_weight(codes, plan)
    if len(shape) != 2 or shape[1] != K:
        raise RuntimeError(f"x must be rows of {K}, got {tuple(shape)}")
    if activation_bits != 16 and activation_bits != 4:
        raise ValueError(f"activation_bits must be 4 or 16, got {activation_bits}")
    R = shape[0]
    grouped = plan_bytes = 0
    shared = 1
    if plan is None:
        if M is not None and M != R:
            raise RuntimeError(f"{M} rows of one weight's, got {R}: without a plan no rows are shared")
        M = R
    else:
        M = R if M is None else M
        grouped, plan_bytes = 1, plan.numel()
        if activation_bits != 16:
            raise RuntimeError("experts' rows are multiplied in 16 bits or more")
        if M != R:
            if R == 0 or M % R:
                raise RuntimeError(f"{M} rows do not share {R} rows of x evenly")
            shared = M // R
    if bias is not None:
        bias = _mx4_bias(bias, dtype, E, N, plan is not None)
    if grouped:
        _mx4_plan(plan, M, E)
    with on(dev):
        y = x.new_empty((M, N))
        if M == 0 or N == 0:
            return y
        x, ldx = _rows(x, K)
        xp = x.data_ptr()
        scratch = _scratch("rq_mx4_linear_scratch_size", dev, code, M, K, N, E, shared, grouped, activation_bits, 0, ldx,
                           xp % 16 == 0)
        nat.call("rq_mx4_linear", xp, code, M, K, ldx, shared, None if plan is None else plan.data_ptr(), plan_bytes,
                 codes.data_ptr(), scales.data_ptr(), E, N, None if bias is None else bias.data_ptr(), activation_bits,
                 y.data_ptr(), N, None if scratch is None else scratch.data_ptr(), 0 if scratch is None else scratch.numel(),
                 nat.stream_handle(dev))
    return y


def mx4_linear_dx(dy: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, K: int, *, plan: Optional[torch.Tensor] = None,
                  shared: int = 1) -> torch.Tensor:
    """dx[t] = sum of dy[r] W[e] over the `shared` rows r of t: mx4_linear's gradient by x.
    dy [M, N]; dx [M / shared, K] in its dtype."""
    _check_mx4(codes, scales, K)
    return _mx4_linear_dx(dy, codes, scales, K, plan, shared)


def _mx4_linear_dx(dy, codes, scales, K, plan, shared):
    """mx4_linear_dx on codes and scales that fit."""
    nat.require_gpu(dy, codes, scales, plan)
    E, N = _mx4_weight(codes, plan)
    if dy.dim() != 2 or dy.shape[1] != N:
        raise RuntimeError(f"dY must be rows of {N}, got {tuple(dy.shape)}")
    M = dy.shape[0]
    if shared < 1 or M % shared or (plan is None and shared != 1):
        raise RuntimeError(f"{M} rows are not {shared} for each row of x")
    if plan is not None:
        _mx4_plan(plan, M, E)
    return _mx4_dx(dy, codes, scales, K, E, N, plan, shared)


def _mx4_dx(dy, codes, scales, K, E, N, plan, shared):
    """mx4_linear_dx of operands that are known to fit (a backward pass's, which autograd has checked)."""
    dev = dy.device
    code = nat.dtype_code(dy.dtype)
    M = dy.shape[0]
    with on(dev):
        dx = dy.new_empty((M // shared, K))
        if M == 0:
            return dx
        if N == 0:
            return dx.zero_()
        dy, lddy = _rows(dy, N)
        dp = dy.data_ptr()
        scratch = _scratch("rq_mx4_linear_scratch_size", dev, code, M, K, N, E, shared, plan is not None, 16, 1, lddy, dp % 16 == 0)
        nat.call("rq_mx4_linear_dx", dp, code, M, N, lddy, None if plan is None else plan.data_ptr(),
                 0 if plan is None else plan.numel(), codes.data_ptr(), scales.data_ptr(), E, K, shared, dx.data_ptr(), K,
                 scratch.data_ptr(), scratch.numel(), nat.stream_handle(dev))
    return dx
