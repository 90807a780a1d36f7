"""MXFP4 linears at their edges: outputs within larger rows, tiles that are split, long contractions, many experts,
gradients of every layout, refusals, graphs side by side, and a block of routed experts that trains and serves."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from rocm_qlora import (ExpertRows, LoRALinear, MXFP4Experts, MXFP4Linear, MXFP4Tensor, dequantize_mxfp4, mxfp4_expert_linear,
                        mxfp4_linear, ops, quantize_mxfp4)
from rocm_qlora import _native as nat
from test_mxfp4_gpu import check, check_experts, check_linear, routes, rows, weight

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,K,N", [(4096, 256, 4100), (3900, 320, 4200), (2300, 128, 7700)])
def test_tiles_past_the_last_whole_round(dev, M, K, N, dtype):
    """Counts of tiles just above a multiple of the compute units, with a last tile of few rows."""
    w, vals = weight(N, K, dev)
    check_linear(rows(M, K, dtype, dev), w, vals, rows(1, N, dtype, dev)[0])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,K,N", [(4096, 512, 4100), (2300, 1100, 7700), (3900, 640, 4200)])
def test_tiles_past_the_last_whole_round_4_bit_activations(dev, M, K, N, dtype):
    """The same for both operands in 4 bits; lengths of half a step among them."""
    w, vals = weight(N, K, dev)
    check_linear(rows(M, K, dtype, dev), w, vals, rows(1, N, dtype, dev)[0], bits=4)


@pytest.mark.parametrize("M,K,N", [(2048, 8500, 100), (2000, 8704, 130)])
def test_gradient_tiles_past_the_last_whole_round(dev, M, K, N):
    w, vals = weight(N, K, dev)
    dy = rows(M, N, BF16, dev)
    d64 = dy.double().cpu()
    check(ops.mx4_linear_dx(dy, w.codes, w.scales, K), d64 @ vals, N, d64.abs() @ vals.abs())


def test_expert_tiles_past_the_last_whole_round(dev):
    check_experts(rows(2048, 256, BF16, dev), routes(2048, 2, 5, 2, skew=0.5), 5, 256, 4200, dev)


@pytest.mark.parametrize("M", [2, 100])
def test_long_contractions_and_wide_outputs(dev, M):
    for K, N in ((1 << 18, 33), (64, 1 << 17)):
        w, vals = weight(N, K, dev)
        check_linear(rows(M, K, BF16, dev), w, vals, dy=rows(M, N, BF16, dev))


@pytest.mark.parametrize("T,k,n", [(1, 1, 1024), (40, 8, 1024), (2000, 2, 1024)])
def test_many_experts(dev, T, k, n):
    g = torch.Generator().manual_seed(T)
    check_experts(rows(T, 160, BF16, dev), torch.randint(0, n, (T, k), generator=g, dtype=torch.int32), n, 160, 48, dev)


# ---- rows behind the results are left as they were ------------------------------------
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("M,K,N", [(3, 256, 37), (40, 512, 100), (130, 640, 301), (600, 1024, 1030), (2500, 512, 2061)])
def test_outputs_within_larger_rows(dev, M, K, N, dtype, bits):
    w, _ = weight(N, K, dev)
    x = rows(M, K, dtype, dev)
    want = mxfp4_linear(x, w, activation_bits=bits)
    code = nat.dtype_code(dtype)
    wide = torch.full((M + 2, N + 5), -7.0, dtype=dtype, device=dev)
    y = wide[1:M + 1, 2:N + 2]
    scratch = ops._scratch("rq_mx4_linear_scratch_size", dev, code, M, K, N, 1, 1, 0, bits, 0, K, 1)
    ws = (None, 0) if scratch is None else (scratch.data_ptr(), scratch.numel())
    nat.call("rq_mx4_linear", x.data_ptr(), code, M, K, K, 1, None, 0, w.codes.data_ptr(), w.scales.data_ptr(), 1, N, None, bits,
             y.data_ptr(), N + 5, *ws, nat.stream_handle(dev))
    assert torch.equal(y, want)
    y.fill_(-7.0)
    assert bool((wide == -7.0).all())
    dy = rows(M, N, dtype, dev, 5)
    dwant = ops.mx4_linear_dx(dy, w.codes, w.scales, K)
    wide = torch.full((M + 2, K + 5), -7.0, dtype=dtype, device=dev)
    dx = wide[1:M + 1, 2:K + 2]
    scratch = ops._scratch("rq_mx4_linear_scratch_size", dev, code, M, K, N, 1, 1, 0, 16, 1, N, 1)
    nat.call("rq_mx4_linear_dx", dy.data_ptr(), code, M, N, N, None, 0, w.codes.data_ptr(), w.scales.data_ptr(), 1, K, 1,
             dx.data_ptr(), K + 5, scratch.data_ptr(), scratch.numel(), nat.stream_handle(dev))
    assert torch.equal(dx, dwant)
    dx.fill_(-7.0)
    assert bool((wide == -7.0).all())


# ---- gradients ------------------------------------------------------------------------
def test_gradients_of_other_layouts(dev):
    """dY broadcast, transposed and strided; x broadcast over rows, shared by two layers, or without a gradient."""
    M, K, N = 90, 200, 150
    w, vals = weight(N, K, dev)
    x = rows(M, K, BF16, dev).requires_grad_(True)
    for dy in (torch.ones(1, 1, dtype=BF16, device=dev).expand(M, N), rows(N, M, BF16, dev).t(), rows(M, 2 * N, BF16, dev)[:, ::2],
               rows(1, N, BF16, dev).expand(M, N)):
        (dx,) = torch.autograd.grad(mxfp4_linear(x, w), x, dy)
        d64 = dy.double().cpu()
        check(dx, d64 @ vals, N, d64.abs() @ vals.abs())
    one = rows(1, K, FP32, dev).requires_grad_(True)
    dy = rows(M, N, FP32, dev)
    (dx,) = torch.autograd.grad(mxfp4_linear(one.expand(M, K), w), one, dy)
    d64 = dy.double().cpu()
    # autograd's own fp32 sum over the rows comes on top
    check(dx, (d64 @ vals).sum(0, keepdim=True), N + M, (d64.abs() @ vals.abs()).sum(0, keepdim=True))
    with torch.inference_mode():
        y = mxfp4_linear(x.detach(), w)
    assert not y.requires_grad and torch.equal(y, mxfp4_linear(x, w).detach())
    assert not mxfp4_linear(x.detach(), w).requires_grad


def test_second_gradients_are_refused(dev):
    w, _ = weight(48, 64, dev)
    x = rows(8, 64, FP32, dev).requires_grad_(True)
    (dx,) = torch.autograd.grad(mxfp4_linear(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# ---- refusals -----------------------------------------------------------------------
def test_refusals(dev):
    w, _ = weight(48, 64, dev)
    we, _ = weight(48, 64, dev, lead=(3,))
    x = rows(8, 64, BF16, dev)
    r = ExpertRows(routes(8, 2, 3).to(dev), 3)
    with pytest.raises(TypeError):
        mxfp4_linear(x.double(), w)
    with pytest.raises(RuntimeError, match="bias"):
        mxfp4_linear(x, w, torch.zeros(47, device=dev))
    with pytest.raises(RuntimeError):
        mxfp4_linear(x, w, torch.zeros(48))  # off the GPU
    with pytest.raises(RuntimeError):
        mxfp4_linear(x, w.to("cpu"))
    with pytest.raises(ValueError, match="activation_bits"):
        mxfp4_linear(x, w, activation_bits=8)
    with pytest.raises(RuntimeError):
        mxfp4_linear(x, we)
    with pytest.raises(RuntimeError, match="bias"):
        mxfp4_expert_linear(x, we, r, torch.zeros(48, device=dev))
    with pytest.raises(RuntimeError, match="by expert"):
        ops.mx4_linear(x[:4], we.codes, we.scales, 64, plan=r.plan, M=8)
    with pytest.raises(RuntimeError, match="by expert"):
        ops.mx4_linear(x, we.codes, we.scales, 64, plan=r.plan.clone(), M=16)
    with pytest.raises(RuntimeError, match="evenly"):
        ops.mx4_linear(x[:3], we.codes, we.scales, 64, plan=r.plan, M=16)
    with pytest.raises(RuntimeError, match="16 bits"):
        ops.mx4_linear(x, we.codes, we.scales, 64, plan=r.plan, M=16, activation_bits=4)
    with pytest.raises(RuntimeError, match="rows of 48"):
        ops.mx4_linear_dx(x, w.codes, w.scales, 64)
    with pytest.raises(RuntimeError, match="by expert"):
        ops.mx4_linear_dx(x[:, :48], we.codes, we.scales, 64, plan=r.plan, shared=2)
    # codes that do not begin on 16 bytes
    held = torch.zeros(48 * 64 + 1, dtype=torch.uint8, device=dev)
    with pytest.raises(RuntimeError):
        mxfp4_linear(x, MXFP4Tensor(held[1:].view(48, 64), w.scales, 64))


# ---- graphs side by side -------------------------------------------------------------
def test_two_graphs_at_once(dev):
    """Two graphs of the same weights, replayed at the same time on streams of their own and in turn with eager calls."""
    K, N, n, T = 640, 384, 4, 300
    w, _ = weight(N, K, dev)
    we, _ = weight(N, K, dev, lead=(n,))

    def made(seed):
        x, dy = rows(T, K, BF16, dev, seed), rows(2 * T, N, BF16, dev, seed + 1)
        ids = routes(T, 2, n, seed).to(dev).to(torch.int32)

        def work():
            r = ExpertRows(ids, n)
            return [mxfp4_linear(x, w), mxfp4_linear(x[:4], w), mxfp4_linear(x, w, activation_bits=4), mxfp4_expert_linear(x, we, r),
                    ops.mx4_linear_dx(dy[:T], w.codes, w.scales, K),
                    ops.mx4_linear_dx(dy, we.codes, we.scales, K, plan=r.plan, shared=2)]

        work()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = work()
        return graph, held, work

    sets = [made(10), made(20)]
    streams = [torch.cuda.Stream() for _ in sets]
    for i in range(3):
        for _, held, _ in sets:
            for t in held:
                t.zero_()
        torch.cuda.synchronize()
        for (graph, _, _), s in zip(sets, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, held, work in sets:
            got = [t.clone() for t in held]
            assert all(torch.equal(a, b) for a, b in zip(got, work())), i


def test_a_captured_backward_pass(dev):
    """Forward and backward pass by autograd in one graph, its leaf made within it, replayed on other inputs."""
    K, N, n, T = 384, 300, 4, 140
    w, _ = weight(N, K, dev)
    we, _ = weight(N, K, dev, lead=(n,))
    x, dy = rows(T, K, BF16, dev), rows(2 * T, N, BF16, dev)
    ids = routes(T, 2, n, 1).to(dev).to(torch.int32)

    def step():
        leaf = x.detach().requires_grad_(True)
        y, z = mxfp4_linear(leaf, w), mxfp4_expert_linear(leaf, we, ExpertRows(ids, n))
        (dx,) = torch.autograd.grad((y, z), leaf, (dy[:T], dy))
        return y.detach(), z.detach(), dx

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = step()
    for i in range(3):
        x.copy_(rows(T, K, BF16, dev, 60 + i))
        dy.copy_(rows(2 * T, N, BF16, dev, 70 + i))
        ids.copy_(routes(T, 2, n, 80 + i).to(dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i


def test_threads_at_once(dev):
    """Calls and backward passes of three threads on streams of their own, the weights shared."""
    K, N, n, T = 384, 300, 4, 130
    w, _ = weight(N, K, dev)
    we, _ = weight(N, K, dev, lead=(n,))

    def work(seed):
        x = rows(T, K, BF16, dev, seed).requires_grad_(True)
        ids = routes(T, 2, n, seed).to(dev)
        outs = []
        for _ in range(10):
            y, z = mxfp4_linear(x, w), mxfp4_expert_linear(x, we, ExpertRows(ids, n))
            outs = [y, z, *torch.autograd.grad((y, z), x, (torch.ones_like(y), torch.ones_like(z)))]
        return [t.detach() for t in outs]

    want = [work(s) for s in range(3)]
    torch.cuda.synchronize()

    def on_own_stream(seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = work(seed)
        torch.cuda.synchronize()
        return got

    with ThreadPoolExecutor(3) as pool:
        for a, b in zip(want, pool.map(on_own_stream, range(3))):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


# ---- a block of routed experts ----------------------------------------------------------
class Block(torch.nn.Module):
    """x + experts(q(x)): a projection with an adapter, and experts of two products whose results are multiplied and
    projected back; the k results of a token are added with its weights."""

    def __init__(self, q, up, gate, down, rank):
        super().__init__()
        self.q = LoRALinear(q, r=rank, lora_alpha=rank)
        self.up, self.gate, self.down = up, gate, down

    def forward(self, x, ids, share):
        r = ExpertRows(ids, self.up.n)
        h = self.q(x)
        a = torch.relu(self.gate(h, r)) * self.up(h, r)
        y = self.down(a, r)
        return x + (y.view(*ids.shape, -1) * share.unsqueeze(-1)).sum(1)


def whole(shape, most, seed, step=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).float() * step


def block(dev, n, D, F, seed=0):
    """Weights of halves and whole numbers that MXFP4 holds exactly, few of them not zero."""
    def some(shape, s):
        return whole(shape, 2, s, 0.5) * (torch.rand(shape, generator=torch.Generator().manual_seed(s + 1)) < 0.2)
    q = torch.nn.Linear(D, D, bias=True)
    q.weight.data, q.bias.data = some((D, D), seed + 2), whole((D,), 2, seed + 4)
    ws = [some(s, seed + 10 + 2 * i).to(dev) for i, s in enumerate([(n, F, D), (n, F, D), (n, D, F)])]
    held = [MXFP4Experts.from_weights(w) for w in ws]
    for w, e in zip(ws, held):
        assert torch.equal(dequantize_mxfp4(MXFP4Tensor(e.weight_quant, e.weight_scales, w.shape[2]), FP32), w)
    m = Block(MXFP4Linear.from_linear(q.to(dev)), *held, rank=4).to(dev)
    m.q.lora_A.data = whole((4, D), 1, seed + 20).to(dev)
    m.q.lora_B.data = whole((D, 4), 1, seed + 21, 0.5).to(dev)
    return m, q.weight.detach().double().cpu(), q.bias.detach().double().cpu(), [w.double().cpu() for w in ws]


def plain_block(x, ids, share, q, b, ws, A, B):
    h = x @ q.t() + b + (x @ A.t()) @ B.t()
    T, k = ids.shape
    y = torch.zeros(T, k, x.shape[1], dtype=torch.float64)
    top = 0.0
    for j in range(k):
        rows_ = []
        for t in range(T):
            e = int(ids[t, j])
            if not 0 <= e < ws[0].shape[0]:
                rows_.append(torch.zeros(x.shape[1], dtype=torch.float64))
                continue
            a = torch.relu(ws[1][e] @ h[t]) * (ws[0][e] @ h[t])
            top = max(top, float((ws[2][e].abs() @ a.detach().abs()).max()))
            rows_.append(ws[2][e] @ a)
        y = y + torch.nn.functional.one_hot(torch.tensor(j), k).view(1, k, 1) * torch.stack(rows_).unsqueeze(1)
    return x + (y * share.unsqueeze(-1)).sum(1), top


@pytest.mark.parametrize("T", [5, 80])
def test_a_block_trains_exactly(dev, T):
    """On fp32 rows of whole numbers every product and sum of the block is exact, so its results and gradients are
    those of the formulas, bit for bit."""
    n, D, F, k = 4, 96, 160, 2
    m, q, b, ws = block(dev, n, D, F)
    ids = routes(T, k, n, 3, missing=True)
    x, share, dy = whole((T, D), 1, 30), whole((T, k), 2, 31, 0.5), whole((T, D), 1, 32)
    ref = [t.double().cpu().requires_grad_(True) for t in (x, share, m.q.lora_A.detach(), m.q.lora_B.detach())]
    want, top = plain_block(ref[0], ids, ref[1], q, b, ws, ref[2], ref[3])
    want.backward(dy.double())
    # in units of 2^-8, with room for a token's two places: below fp32's 24 bits
    assert top * 2 ** 8 < 2 ** 24 and all(float(t.grad.abs().max()) * 2 ** 7 < 2 ** 24 for t in ref)
    assert all(torch.equal(t.grad, t.grad.float().double()) for t in ref)
    xg, sg = x.to(dev).requires_grad_(True), share.to(dev).requires_grad_(True)
    y = m(xg, ids.to(dev), sg)
    y.backward(dy.to(dev))
    assert torch.equal(y.detach().double().cpu(), want.detach())
    for got, t in zip((xg, sg, m.q.lora_A, m.q.lora_B), ref):
        assert torch.equal(got.grad.double().cpu(), t.grad)
    # served a token at a time
    with torch.no_grad():
        for t in range(min(T, 6)):
            one = m(xg[t:t + 1], ids[t:t + 1].to(dev), sg[t:t + 1])
            assert torch.equal(one.double().cpu(), want[t:t + 1].detach())


def test_a_block_serves_from_a_graph(dev):
    """One token captured, its router and all, and replayed on other tokens."""
    n, D, F, k = 8, 256, 384, 2
    m, _, _, _ = block(dev, n, D, F, 5)
    m = m.to(BF16).eval()
    router = torch.nn.Linear(D, n, bias=False).to(dev).to(BF16)
    x = rows(1, D, BF16, dev)

    def step():
        with torch.no_grad():
            p, ids = router(x).float().topk(k, dim=1)
            return m(x, ids, p.softmax(1).to(BF16))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for i in range(4):
        x.copy_(rows(1, D, BF16, dev, 50 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, step()), i
