"""The MXFP4 codec, linears and experts' linears against their definitions in 64 bits.  Codes,
scales and values are exact; results are within the roundings that mxfp4_oracle.tolerance counts."""
import numpy as np
import pytest
import torch

import mxfp4_oracle as oracle
from rocm_qlora import (ExpertRows, LoRALinear, MXFP4Experts, MXFP4Linear, MXFP4Tensor, dequantize_mxfp4, mxfp4_expert_linear,
                        mxfp4_linear, ops, quantize_mxfp4)

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


# ---- codec ------------------------------------------------------------------------
def check_codec(x):
    t = quantize_mxfp4(x)
    K = x.shape[-1]
    codes, scales, vals = oracle.quantize(x.reshape(-1, K))
    assert t.shape == x.shape
    assert np.array_equal(t.scales.reshape(-1, t.scales.shape[-1]).cpu().numpy().astype(np.int64), scales)
    got = oracle.unpack(t.codes.reshape(-1, t.codes.shape[-1]))
    nan = np.repeat(scales == 255, 32, axis=1)
    assert np.array_equal(got[~nan], codes[~nan])
    for dtype in (BF16, FP32, FP16):
        back = dequantize_mxfp4(t, dtype)
        assert back.dtype == dtype and back.shape == x.shape
        # exact in bf16 and fp32, one rounding in fp16
        want = torch.from_numpy(vals[:, :K]).to(dtype).double().numpy()
        have = back.reshape(-1, K).double().cpu().numpy()
        assert np.array_equal(have, want, equal_nan=True)
        assert np.array_equal(np.signbit(have[~np.isnan(have)]), np.signbit(want[~np.isnan(want)]))
    return t


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 31), (2, 33), (5, 48), (4, 127), (7, 129), (33, 1001), (9, 4096),
                                 (300, 256), (2, 9000)])
def test_codec(dev, M, K, dtype):
    g = torch.Generator().manual_seed(M * K)
    x = torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    check_codec(x.to(dtype).to(dev))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_codec_ties_and_extremes(dev, dtype):
    """Every middle between two codes, both signs, at scales from the type's least to its largest."""
    fin = torch.finfo(dtype)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.0, 6.0, 7.5, 0.5, 1.0, 1.5, 3.0, 4.0], dtype=torch.float64)
    block = torch.cat([mids, -mids])
    rows = []
    for e in (-126, -100, -24, -14, -3, 0, 5, 12, 100, 124):
        r = block * 2.0 ** e
        if r.abs().max() <= fin.max:
            rows.append(r)
    x = torch.stack(rows).to(dtype)
    nudged = torch.stack([x, torch.nextafter(x, torch.full_like(x, float("inf"))), torch.nextafter(x, -torch.full_like(x, float("inf")))])
    check_codec(nudged.reshape(-1, 32).to(dev))
    edge = torch.tensor([fin.max, -fin.max, fin.tiny, fin.smallest_normal, -fin.smallest_normal, 0.0, -0.0, 1.0], dtype=dtype)
    sub = torch.full((8, 32), 0.0, dtype=dtype)
    sub[:, 3] = edge
    sub[:, 17] = edge.flip(0) / 3
    check_codec(sub.to(dev))
    least = torch.zeros(4, 64, dtype=dtype)
    least[:, :8] = torch.finfo(dtype).smallest_normal * fin.eps * torch.arange(8).to(dtype)
    check_codec(least.to(dev))


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_codec_nan_blocks(dev, dtype, bad):
    x = torch.randn(3, 100, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[1, 40] = bad
    x[2, 99] = bad
    t = check_codec(x.to(dev))
    assert int((t.scales == 255).sum()) == 2


def test_codec_layouts(dev):
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    whole = quantize_mxfp4(x)
    for v in (x[:, 1:], x[::2], x[:, :256], x.reshape(2, 3, 300), x.t().contiguous().t(), x[:1].expand(4, 300)):
        check_codec(v)
    on_cpu = quantize_mxfp4(x.cpu())
    assert on_cpu.codes.device.type == "cpu" and torch.equal(on_cpu.codes, whole.codes.cpu())
    assert torch.equal(dequantize_mxfp4(on_cpu), dequantize_mxfp4(whole).cpu())
    assert quantize_mxfp4(x[:0]).shape == (0, 300)
    assert dequantize_mxfp4(quantize_mxfp4(x[:0])).shape == (0, 300)


# ---- linears -----------------------------------------------------------------------
def weight(N, K, dev, seed=0, lead=()):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(*lead, N, K, generator=g) * 0.02 * torch.exp(torch.randn(*lead, N, 1, generator=g))
    t = quantize_mxfp4(w.to(dev))
    return t, oracle.held(t.codes, t.scales, K)


def rows(M, K, dtype, dev, seed=1):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(seed + 17 * M + K)).to(dtype).to(dev)


def check(got, want, terms, size):
    assert got.shape == want.shape
    off = (got.detach().double().cpu() - want).abs()
    tol = oracle.tolerance(got.dtype, want, terms, size)
    assert bool((off <= tol).all()), f"off by {float((off / tol).max())} of the tolerance at {np.unravel_index(int((off / tol).argmax()), off.shape)}"


def check_linear(x, w, vals, bias=None, bits=16, dy=None):
    K, N = w.K, vals.shape[0]
    x64 = x.detach().double().cpu().reshape(-1, K)
    if bits == 4:
        x64 = torch.from_numpy(oracle.quantize(x.detach().reshape(-1, K))[2][:, :K])
    want, size = x64 @ vals.t(), x64.abs() @ vals.abs().t()
    if bias is not None:
        want, size = want + bias.double().cpu(), size + bias.double().cpu().abs()
    y = mxfp4_linear(x, w, bias, activation_bits=bits)
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], N)
    check(y.reshape(-1, N), want, K, size)
    if dy is not None:
        xg = x.detach().requires_grad_(True)
        yg = mxfp4_linear(xg, w, bias, activation_bits=bits)
        assert torch.equal(yg, y)
        (dx,) = torch.autograd.grad(yg, xg, dy)
        d64 = dy.double().cpu().reshape(-1, N)
        assert dx.shape == x.shape and dx.dtype == x.dtype
        check(dx.reshape(-1, K), d64 @ vals, N, d64.abs() @ vals.abs())


SIZES = [(1, 128, 16), (1, 4096, 4096), (2, 31, 7), (3, 1, 1), (5, 130, 100), (16, 256, 257), (17, 1000, 48), (33, 333, 129),
         (64, 512, 64), (65, 128, 256), (66, 64, 300), (100, 1000, 513), (129, 640, 260), (200, 96, 1030), (256, 2048, 256),
         (300, 129, 64), (513, 1024, 700), (1000, 257, 1000)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(dev, M, K, N, dtype):
    w, vals = weight(N, K, dev)
    bias = rows(1, N, dtype, dev)[0] if (M + N) % 2 else None
    check_linear(rows(M, K, dtype, dev), w, vals, bias, dy=rows(M, N, dtype, dev, 5))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_4_bit_activations(dev, M, K, N, dtype):
    w, vals = weight(N, K, dev, 3)
    bias = rows(1, N, dtype, dev)[0] if (M + N) % 2 else None
    check_linear(rows(M, K, dtype, dev), w, vals, bias, bits=4, dy=rows(M, N, dtype, dev, 5) if M < 70 else None)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("M,K,N", [(2048, 1024, 1280), (1500, 4096, 2048), (4096, 384, 4200)])
def test_linear_large(dev, M, K, N, dtype):
    """Whole waves of tiles, and tiles' ends."""
    w, vals = weight(N, K, dev, 4)
    check_linear(rows(M, K, dtype, dev), w, vals, dy=rows(M, N, dtype, dev, 5))
    check_linear(rows(M, K, dtype, dev), w, vals, bits=4)


@pytest.mark.parametrize("M", [3, 40, 100, 400])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_linear_layouts(dev, M, dtype):
    K, N = 256, 192
    w, vals = weight(N, K, dev, 6)
    wide = rows(2 * M, K + 8, dtype, dev)
    for x in (wide[:M, 1:K + 1], wide[:M, 8:], wide[::2, :K], wide[:M, :K].t().contiguous().t(), wide[:1, :K].expand(M, K),
              wide[:2 * (M // 2), :K].reshape(2, M // 2, K)):
        dy = rows(x.numel() // K, N + 3, dtype, dev, 9)[:, 3:].reshape(*x.shape[:-1], N)
        check_linear(x, w, vals, dy=dy)
        check_linear(x, w, vals, bits=4)
    # a gradient that is broadcast, as that of a sum
    x = wide[:M, :K].detach().requires_grad_(True)
    mxfp4_linear(x, w).sum().backward()
    check(x.grad, vals.sum(0).expand(M, K), N, vals.abs().sum(0).expand(M, K))


@pytest.mark.parametrize("M", [2, 70, 300])
def test_linear_not_a_number(dev, M):
    """An infinity or a NaN in a row, or a NaN block of the weight, reaches what it is a factor of and nothing else."""
    K, N = 256, 70
    w, vals = weight(N, K, dev, 7)
    w.scales[5, 3] = 255
    for dtype in (BF16, FP32):
        x = rows(M, K, dtype, dev)
        clean = mxfp4_linear(x, w)
        assert bool(clean[:, 5].isnan().all()) and not bool(clean[:, :5].isnan().any()) and not bool(clean[:, 6:].isnan().any())
        x[1, 9] = float("nan")
        y = mxfp4_linear(x, w)
        assert bool(y[1].isnan().all())
        assert torch.equal(y[0], clean[0]) or bool(clean[0].isnan().any()) and torch.equal(y[0].nan_to_num(), clean[0].nan_to_num())
        x[1, 9] = float("inf")
        y = mxfp4_linear(x, w)
        assert not bool(y[1].isfinite().any()) and bool(y[0, :5].isfinite().all())
        y4 = mxfp4_linear(x, w, activation_bits=4)
        assert bool(y4[1].isnan().all()) and bool(y4[0, :5].isfinite().all())
        dy = rows(M, N, dtype, dev, 3)
        dx = ops.mx4_linear_dx(dy, w.codes, w.scales, K)
        assert bool(dx[:, 96:128].isnan().all()) and bool(dx[:, :96].isfinite().all()) and bool(dx[:, 128:].isfinite().all())


def test_linear_fp32_is_exact_in_its_factors(dev):
    """fp32 rows lose no bit to the three parts: one product a sum, largest and smallest magnitudes."""
    K, N = 128, 16
    t = MXFP4Tensor(torch.zeros(N, K // 2, dtype=torch.uint8, device=dev), torch.full((N, K // 32), 127, dtype=torch.uint8, device=dev), K)
    t.codes[:, 0] = 2  # 1.0 times the first value
    for M in (4, 200):
        x = torch.zeros(M, K, device=dev)
        x[:, 0] = torch.randn(M, generator=torch.Generator().manual_seed(3)).to(dev) * 2.0 ** torch.linspace(-100, 126, M).to(dev)
        x[0, 0] = torch.finfo(FP32).max
        assert torch.equal(mxfp4_linear(x, t), x[:, :1].expand(M, N))


def test_linear_empty(dev):
    w, _ = weight(40, 200, dev)
    x = torch.empty(0, 200, dtype=BF16, device=dev, requires_grad=True)
    y = mxfp4_linear(x, w)
    assert y.shape == (0, 40)
    y.sum().backward()
    assert x.grad.shape == (0, 200)


# ---- experts -----------------------------------------------------------------------
def check_experts(x, ids, n, K, N, dev, bias=None, shared=True, train=True, seed=0):
    w, vals = weight(N, K, dev, 11 + seed, (n,))
    T, k = ids.shape
    r = ExpertRows(ids.to(dev), n)
    x64 = x.detach().double().cpu()
    x64 = x64.repeat_interleave(k, 0) if shared else x64
    flat = ids.reshape(-1)
    want, size = torch.zeros(T * k, N, dtype=torch.float64), torch.zeros(T * k, N, dtype=torch.float64)
    for e in range(n):
        on = flat == e
        want[on], size[on] = x64[on] @ vals[e].t(), x64[on].abs() @ vals[e].abs().t()
        if bias is not None:
            b = bias[e].double().cpu()
            want[on] += b
            size[on] += b.abs()
    xg = x.detach().requires_grad_(train)
    y = mxfp4_expert_linear(xg, w, r, bias)
    assert y.dtype == x.dtype
    check(y, want, K, size)
    none = (flat < 0) | (flat >= n)
    assert not bool(y.detach()[none.to(dev)].any())
    if train:
        dy = rows(T * k, N, x.dtype, dev, 21)
        (dx,) = torch.autograd.grad(y, xg, dy)
        d64 = dy.double().cpu()
        dw, ds = torch.zeros(T * k, K, dtype=torch.float64), torch.zeros(T * k, K, dtype=torch.float64)
        for e in range(n):
            on = flat == e
            dw[on], ds[on] = d64[on] @ vals[e], d64[on].abs() @ vals[e].abs()
        if shared:
            dw, ds = dw.view(T, k, K).sum(1), ds.view(T, k, K).sum(1)
        check(dx, dw, N + k, ds)


def routes(T, k, n, seed=0, skew=1.5, missing=False):
    g = torch.Generator().manual_seed(seed)
    p = torch.arange(1, n + 1, dtype=torch.float64) ** -skew
    ids = torch.stack([torch.multinomial(p, k, generator=g) for _ in range(T)]) if T else torch.zeros(0, k, dtype=torch.int64)
    if missing:
        ids[torch.rand(T, k, generator=g) < 0.3] = -1
        ids[torch.rand(T, k, generator=g) < 0.1] = n + 3
    return ids.to(torch.int32 if seed % 2 else torch.int64)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,k,n,K,N", [(1, 1, 1, 128, 64), (1, 2, 8, 256, 40), (8, 2, 64, 512, 96), (5, 3, 4, 100, 33), (30, 4, 6, 256, 300),
                                       (64, 1, 3, 333, 130), (100, 2, 5, 640, 257), (200, 4, 4, 256, 512), (300, 8, 16, 128, 260),
                                       (700, 2, 3, 384, 129)])
def test_experts(dev, T, k, n, K, N, dtype):
    ids = routes(T, k, n, T + k)
    bias = rows(n, N, dtype, dev) if T % 2 == 0 else None
    check_experts(rows(T, K, dtype, dev), ids, n, K, N, dev, bias)
    check_experts(rows(T * k, K, dtype, dev), ids, n, K, N, dev, None, shared=k == 1)


@pytest.mark.parametrize("T", [3, 90, 400])
def test_experts_rows_without_one(dev, T):
    check_experts(rows(T, 256, BF16, dev), routes(T, 2, 5, T, missing=True), 5, 256, 140, dev, rows(5, 140, BF16, dev))
    check_experts(rows(T, 256, BF16, dev), torch.full((T, 2), -1), 5, 256, 140, dev, rows(5, 140, BF16, dev))
    # all on the last one, or the same one twice
    check_experts(rows(T, 256, BF16, dev), torch.full((T, 2), 4), 5, 256, 140, dev)


def test_experts_layouts(dev):
    K, N, n, T, k = 256, 96, 4, 150, 2
    ids = routes(T, k, n, 3)
    wide = rows(2 * T, K + 8, BF16, dev)
    for x in (wide[:T, 1:K + 1], wide[:T, 8:], wide[::2, :K], wide[:1, :K].expand(T, K), wide[:T, :K].t().contiguous().t()):
        check_experts(x, ids, n, K, N, dev)


def test_experts_empty(dev):
    w, _ = weight(40, 200, dev, lead=(3,))
    x = torch.empty(0, 200, dtype=BF16, device=dev, requires_grad=True)
    y = mxfp4_expert_linear(x, w, ExpertRows(torch.empty(0, 2, dtype=torch.int32, device=dev), 3))
    assert y.shape == (0, 40)
    y.sum().backward()
    assert x.grad.shape == (0, 200)


def test_rows_past_4_gib(dev):
    """Rows whose offsets do not fit 32 bits, of one weight and of experts."""
    K, N, M = 256, 48, 150
    far = torch.empty(M * (1 << 25), dtype=BF16, device=dev).view(M, 1 << 25)
    x = far[:, :K]
    x.copy_(rows(M, K, BF16, dev))
    near = x.contiguous()
    w, _ = weight(N, K, dev)
    assert torch.equal(mxfp4_linear(x, w), mxfp4_linear(near, w))
    assert torch.equal(mxfp4_linear(x[:20], w), mxfp4_linear(near[:20], w))
    we, _ = weight(N, K, dev, lead=(3,))
    r = ExpertRows(routes(M, 2, 3, 1).to(dev), 3)
    assert torch.equal(mxfp4_expert_linear(x, we, r), mxfp4_expert_linear(near, we, r))
    assert torch.equal(ops.mx4_linear_dx(far[:, :N], w.codes, w.scales, K), ops.mx4_linear_dx(near[:, :N], w.codes, w.scales, K))


# ---- layers, gradients against differences, streams, graphs -----------------------------
def test_layers(dev):
    torch.manual_seed(0)
    lin = torch.nn.Linear(300, 150).to(dev).to(BF16)
    m = MXFP4Linear.from_linear(lin)
    x = rows(20, 300, BF16, dev).view(4, 5, 300)
    t = MXFP4Tensor(m.weight_quant, m.weight_scales, 300)
    assert torch.equal(m(x), mxfp4_linear(x, t, lin.bias.detach()))
    assert torch.equal(m.dequantized_weight(), dequantize_mxfp4(t))
    other = MXFP4Linear(300, 150).to(dev)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.to(BF16)(x), m(x))
    four = MXFP4Linear.from_linear(lin, activation_bits=4)
    assert torch.equal(four(x), mxfp4_linear(x, t, lin.bias.detach(), activation_bits=4))
    lora = LoRALinear(m, r=4)
    torch.nn.init.normal_(lora.lora_B, std=0.02)
    xg = x.detach().requires_grad_(True)
    y = lora(xg)
    y.float().sum().backward()
    assert lora.lora_A.grad is not None and xg.grad.shape == x.shape
    experts = MXFP4Experts.from_weights([torch.nn.Linear(300, 40, device=dev) for _ in range(3)])
    r = ExpertRows(routes(20, 2, 3, 1).to(dev), 3)
    y = experts(x.view(20, 300), r)
    w = MXFP4Tensor(experts.weight_quant, experts.weight_scales, 300)
    assert torch.equal(y, mxfp4_expert_linear(x.view(20, 300), w, r, experts.bias))


@pytest.mark.parametrize("kind", ["linear", "experts"])
def test_gradient_against_differences(dev, kind):
    """The map is linear: f(x + h v) - f(x - h v) = 2 h (dY W) v up to fp32 roundings."""
    K, N, T, k, n = 192, 80, 70, 2, 3
    x = rows(T, K, FP32, dev)
    v = rows(T, K, FP32, dev, 31)
    if kind == "linear":
        w, _ = weight(N, K, dev)
        f = lambda z: mxfp4_linear(z, w)  # noqa: E731
    else:
        w, _ = weight(N, K, dev, lead=(n,))
        r = ExpertRows(routes(T, k, n, 1).to(dev), n)
        f = lambda z: mxfp4_expert_linear(z, w, r)  # noqa: E731
    xg = x.clone().requires_grad_(True)
    y = f(xg)
    c = rows(y.shape[0], N, FP32, dev, 41)
    (dx,) = torch.autograd.grad(y, xg, c)
    with torch.no_grad():
        h = 0.25
        diff = ((f(x + h * v) - f(x - h * v)).double() * c.double()).sum() / (2 * h)
        want = (dx.double() * v.double()).sum()
        # each of the y.numel() outputs is off by (K + 2) 2^-23 of its products' magnitudes at most, which are
        # under |x| + h |v| times the weight's largest column sum; the gradient likewise by (N + 2) 2^-23
        mag = float((f(x.abs() + h * v.abs()).abs().double() * c.abs().double()).sum())
    big = float((x.abs() + h * v.abs()).max()) * K * float(dequantize_mxfp4(w, FP32).abs().max())
    tol = 2 * (K + N + 4) * 2.0 ** -23 * (mag + big * float(c.abs().double().sum())) / (2 * h)
    assert abs(float(diff - want)) <= tol


def test_two_runs_are_equal_and_streams(dev):
    K, N, n = 512, 300, 4
    w, _ = weight(N, K, dev)
    we, _ = weight(N, K, dev, lead=(n,))
    ids = routes(200, 2, n, 1).to(dev)
    x, dy = rows(200, K, BF16, dev), rows(400, N, BF16, dev)

    def work():
        r = ExpertRows(ids, n)
        return [mxfp4_linear(x, w), mxfp4_linear(x[:3], w), mxfp4_linear(x, w, activation_bits=4), mxfp4_linear(x[:9], w, activation_bits=4),
                mxfp4_expert_linear(x, we, r), ops.mx4_linear_dx(dy[:200], w.codes, w.scales, K),
                ops.mx4_linear_dx(dy, we.codes, we.scales, K, plan=r.plan, shared=2)]

    first = work()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(work())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(first, o))


def test_graph_replays(dev):
    """The whole set captured once and replayed on changed inputs, with eager work between."""
    K, N, n, T = 512, 384, 4, 150
    w, _ = weight(N, K, dev)
    we, _ = weight(N, K, dev, lead=(n,))
    x, dy = rows(T, K, BF16, dev), rows(2 * T, N, BF16, dev)
    ids = routes(T, 2, n, 1).to(dev).to(torch.int32)

    def work():
        r = ExpertRows(ids, n)
        t = quantize_mxfp4(x)
        return [t.codes, t.scales, dequantize_mxfp4(t), mxfp4_linear(x, w), mxfp4_linear(x[:5], w), mxfp4_linear(x, w, activation_bits=4),
                mxfp4_expert_linear(x, we, r), ops.mx4_linear_dx(dy[:T], w.codes, w.scales, K),
                ops.mx4_linear_dx(dy, we.codes, we.scales, K, plan=r.plan, shared=2)]

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(3):
        x.copy_(rows(T, K, BF16, dev, 100 + i))
        dy.copy_(rows(2 * T, N, BF16, dev, 200 + i))
        ids.copy_(routes(T, 2, n, 2 * i + 1).to(dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, work())), i
