"""Adapters of many requests: forward, gradients, grouping, layers.

Oracle: the formulas in fp64 on the CPU.  Bounds, with U the unit roundoff of
the dtype (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and |.| sums of absolute products:
a result is rounded once (U |y|); the first product is passed on in two 16-bit
parts (U^2 of the second product's absolute sum; fp16 adds the parts' smallest
step, 2^-24); a sum of n fp32 terms errs by n 2^-24 of its absolute sum."""
import pytest
import torch

from rocm_qlora import LoRALinear, QuantLinear, ops
from rocm_qlora.lora import AdapterRows, MultiLoRALinear, attach_adapters, multi_lora, set_adapter_rows

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}
E32 = 2.0 ** -24


def make(M, K, N, r, n, dtype, dev, seed=0, ids=None):
    g = torch.Generator().manual_seed(seed)
    d = {"x": torch.randn(M, K, generator=g), "base": torch.randn(M, N, generator=g),
         "a": torch.randn(n, r, K, generator=g) / K ** 0.5, "b": torch.randn(n, N, r, generator=g) * 0.2,
         "dy": torch.randn(M, N, generator=g) * 0.1}
    d = {k: v.to(dtype).to(dev) for k, v in d.items()}
    d["s"] = (torch.rand(n, generator=g) * 2 + 0.5).to(dev)
    if ids is None:
        ids = torch.randint(-1, n, (M,), generator=g, dtype=torch.int32)
    d["ids"] = torch.as_tensor(ids, dtype=torch.int32).to(dev)
    return d


def oracle(d, held=None):
    """Values and absolute sums of y, dx, dA, dB in fp64."""
    c = {k: v.detach().double().cpu() for k, v in d.items()}
    x, a, b, s, ids, dy = c["x"], c["a"], c["b"], c["s"], d["ids"].cpu(), c["dy"]
    held = x if held is None else held.double().cpu()
    y, ya = c["base"].clone(), torch.zeros_like(c["base"])
    dx, dxa = torch.zeros_like(x), torch.zeros_like(x)
    da, daa, db, dba = torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(b)
    step = torch.zeros_like(c["base"]), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for i in range(a.shape[0]):
        on = ids == i
        if not bool(on.any()):
            continue
        u, ua = x[on] @ a[i].T, x[on].abs() @ a[i].abs().T
        g, ga = s[i] * (dy[on] @ b[i]), s[i] * (dy[on].abs() @ b[i].abs())
        y[on] += s[i] * (u @ b[i].T)
        ya[on] = s[i] * (ua @ b[i].abs().T)
        dx[on], dxa[on] = g @ a[i], ga @ a[i].abs()
        da[i], daa[i] = g.T @ held[on], ga.T @ held[on].abs()
        db[i], dba[i] = s[i] * dy[on].T @ u, s[i] * dy[on].abs().T @ ua
        step[0][on] = s[i] * b[i].abs().sum(1)
        step[1][on] = a[i].abs().sum(0)
        step[2][i] = held[on].abs().sum(0)
        step[3][i] = s[i] * dy[on].abs().sum(0)[:, None]
    return (y, dx, da, db), (ya, dxa, daa, dba), step


def check(got, want, absum, step, dtype, terms, name):
    got = got.detach().double().cpu()
    half = 0.0 if dtype == FP32 else U[dtype] ** 2
    bound = U[dtype] * want.abs() + (half + terms * E32) * absum + E32 * want.abs()
    if dtype == FP16:
        bound += 2.0 ** -24 * (step + 1)
    err = (got - want).abs()
    assert torch.equal(got.isnan(), want.isnan()), name
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: error {worst:.2f} times its bound"


def run_all(d, rows, bits=16):
    x, a, b = (d[k].detach().clone().requires_grad_(True) for k in ("x", "a", "b"))
    y = multi_lora(x, a, b, d["s"], rows, d["base"], bits)
    dx, da, db = torch.autograd.grad(y, (x, a, b), d["dy"])
    return y, dx, da, db


def check_all(d, got, bits=16):
    held = None
    dtype = d["x"].dtype
    if bits == 8:
        held = ops.act8_dequantize(*ops.act8_quantize(d["x"]), d["x"].shape[1], dtype)
    want, absum, step = oracle(d, held)
    (M, K), N, r = d["x"].shape, d["b"].shape[1], d["a"].shape[1]
    for name, g, w, s, t, n in zip(("y", "dx", "dA", "dB"), got, want, absum, step, (K + r, N + r, N + M, K + M)):
        check(g, w, s, t, dtype, n + 8, f"{name} of {M}x{K}x{N} r={r} n={d['a'].shape[0]} {dtype}")


SHAPES = [
    # M, K, N, r, n
    (1, 64, 64, 8, 1),
    (1, 1, 1, 1, 1),
    (2, 7, 5, 3, 2),
    (8, 512, 256, 16, 4),
    (16, 130, 257, 16, 16),
    (33, 1000, 1501, 10, 3),
    (64, 256, 128, 64, 1),
    (65, 96, 520, 33, 2),
    (129, 515, 640, 48, 5),
    (200, 1024, 1024, 17, 40),
    (257, 320, 72, 65, 3),
    (300, 192, 192, 130, 2),
    (100, 40, 37, 1, 1),
    (130, 700, 705, 3, 2),
    (150, 384, 520, 20, 2),
    (90, 136, 129, 300, 2),
    (70, 512, 384, 512, 1),
    (700, 2049, 300, 32, 3),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K,N,r,n", SHAPES)
def test_forward_and_gradients(dev, M, K, N, r, n, dtype):
    print(f"multi_lora {M}x{K}x{N} r={r} n={n} {dtype}", flush=True)
    d = make(M, K, N, r, n, dtype, dev, seed=M + K)
    check_all(d, run_all(d, AdapterRows(d["ids"], n)))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K,N,r", [(1, 32, 64, 8), (70, 260, 130, 12), (1500, 128, 96, 16), (130, 96, 1024, 64)])
def test_single_adapter_without_grouping(dev, M, K, N, r, dtype):
    d = make(M, K, N, r, 1, dtype, dev, seed=3, ids=torch.zeros(M))
    got = run_all(d, AdapterRows.single(M))
    check_all(d, got)
    # grouped, the same rows in the same order: the same bits but for sums over rows in other chunks
    same = run_all(d, AdapterRows(d["ids"], 1))
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K,N,r,n", [(40, 64, 96, 8, 2), (333, 1001, 130, 12, 3), (600, 512, 256, 40, 1)])
def test_gradients_from_8_bit_checkpoint(dev, M, K, N, r, n, dtype):
    d = make(M, K, N, r, n, dtype, dev, seed=5)
    rows = AdapterRows(d["ids"], n)
    got = run_all(d, rows, bits=8)
    check_all(d, got, bits=8)
    full = run_all(d, rows)
    for i in (0, 1, 3):  # x is read from the codes for dA alone
        assert torch.equal(got[i], full[i])


@pytest.mark.parametrize("ids", [
    [-1] * 70,                                   # no row has an adapter
    [2] * 70,                                    # two adapters have no rows
    [0] * 64 + [2] * 6,                          # one full tile
    [5, -7, 3, 0, 1, 2, 2 ** 30, -2 ** 31] + [1] * 62,  # ids that are no adapter's
    ([0, 1, 2, -1] * 18)[:70],                   # interleaved
])
def test_rows_without_adapters_and_adapters_without_rows(dev, ids):
    d = make(70, 96, 80, 8, 3, BF16, dev, seed=9, ids=torch.tensor(ids))
    y, dx, da, db = got = run_all(d, AdapterRows(d["ids"], 3))
    check_all(d, got)
    none = ~((d["ids"] >= 0) & (d["ids"] < 3))
    assert torch.equal(y[none], d["base"][none])
    assert not dx[none].any()
    for i in range(3):
        if not bool((d["ids"] == i).any()):
            assert not da[i].any() and not db[i].any()


def test_grouping_of_many_rows(dev):
    """Several chunks an adapter (partial sums), adapters of one row, 1024 adapters, int64 ids."""
    g = torch.Generator().manual_seed(1)
    M, n = 5000, 1024
    ids = torch.where(torch.rand(M, generator=g) < 0.7, torch.zeros(M, dtype=torch.int64), torch.randint(-1, n, (M,), generator=g))
    d = make(M, 40, 24, 4, n, FP32, dev, ids=ids.to(torch.int32))
    rows = AdapterRows(ids.to(dev), n)
    check_all(d, run_all(d, rows))
    again = run_all(d, AdapterRows(ids.to(dev), n))
    for a, b in zip(run_all(d, rows), again):
        assert torch.equal(a, b)  # no sum's order is left open


def test_wide_int64_ids_have_no_adapter(dev):
    d = make(3, 32, 32, 4, 2, FP32, dev, ids=[-1, -1, 1])
    rows = AdapterRows(torch.tensor([1 + 2 ** 32, -2 ** 40, 1], device=dev), 2)
    check_all(d, run_all(d, rows))


def test_not_a_number_stays_in_its_rows(dev):
    d = make(80, 64, 48, 8, 2, BF16, dev, ids=[0] * 40 + [1] * 40)
    d["x"][5, 3] = float("nan")
    d["x"][45, 2] = float("inf")
    d["dy"][7, 1] = float("nan")
    y, dx, da, db = run_all(d, AdapterRows(d["ids"], 2))
    bad = torch.zeros(80, dtype=torch.bool, device=dev)
    bad[[5, 45]] = True
    assert bool(torch.isfinite(y[~bad]).all()) and bool(y[5].isnan().all())
    bad[:] = False
    bad[7] = True
    assert bool(torch.isfinite(dx[~bad]).all())
    assert bool(da[0].isnan().any()) and bool(db[0].isnan().any())
    assert not bool(da[1].isnan().any(0).all())  # adapter 1's rows hold no NaN; its infinity shows in one column of dA


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_infinity_of_a_row_stays_one(dev, dtype):
    # one sign throughout, so that the formula's results are infinities, whatever the padded ranks
    for M, r in ((1, 1), (20, 3), (70, 1)):
        d = make(M, 40, 36, r, 1, dtype, dev, ids=[0] * M)
        d["a"], d["b"], d["x"][0, 7] = d["a"].abs() + 0.01, d["b"].abs() + 0.01, float("inf")
        y = multi_lora(d["x"], d["a"], d["b"], d["s"], AdapterRows(d["ids"], 1), d["base"])
        assert bool((y[0] == float("inf")).all()) and bool(torch.isfinite(y[1:]).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strides_and_alignment(dev, dtype):
    M, K, N, r, n = 37, 72, 90, 6, 2
    d = make(M, K, N, r, n, dtype, dev, seed=2)
    rows = AdapterRows(d["ids"], n)
    want = multi_lora(d["x"], d["a"], d["b"], d["s"], rows, d["base"])
    wide = torch.zeros(M, K + 5, dtype=dtype, device=dev)
    wide[:, 3:3 + K] = d["x"]
    wbase = torch.zeros(M, N + 3, dtype=dtype, device=dev)
    wbase[:, 1:1 + N] = d["base"]
    assert torch.equal(multi_lora(wide[:, 3:3 + K], d["a"], d["b"], d["s"], rows, wbase[:, 1:1 + N]), want)
    assert torch.equal(multi_lora(d["x"].t().contiguous().t(), d["a"], d["b"], d["s"], rows, d["base"]), want)
    a_t = d["a"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(multi_lora(d["x"], a_t, d["b"], d["s"], rows, d["base"]), want)
    # in place, into a strided result whose other columns stay
    out = wbase.clone()
    res = ops.multi_lora(d["x"], d["a"], d["b"], d["s"], rows.plan, out[:, 1:1 + N], out[:, 1:1 + N])
    assert torch.equal(res, want) and torch.equal(out[:, :1], wbase[:, :1]) and torch.equal(out[:, 1 + N:], wbase[:, 1 + N:])
    # without a base: the term alone
    zero = multi_lora(d["x"], d["a"], d["b"], d["s"], rows, torch.zeros_like(d["base"]))
    assert torch.equal(multi_lora(d["x"], d["a"], d["b"], d["s"], rows), zero)
    # leading dimensions
    x3, b3 = d["x"][:36].view(4, 9, K), d["base"][:36].view(4, 9, N)
    r3 = AdapterRows(d["ids"][:36].view(4, 9), n)
    assert torch.equal(multi_lora(x3, d["a"], d["b"], d["s"], r3, b3), want[:36].view(4, 9, N))


def test_more_than_2_to_the_31_values(dev):
    """Results and dY of more elements than 32 bits count: the first and the last rows' results,
    and the gradients of a dY that is zero before the last rows."""
    M, K, N, r, n, last = 33000, 40, 65568, 8, 2, 50
    d = make(last + 20, K, N, r, n, BF16, dev, seed=9)
    held = torch.cat([torch.arange(20, device=dev), torch.arange(M - last, M, device=dev)])
    big = dict(d, x=torch.randn(M, K, device=dev).to(BF16), ids=torch.randint(-1, n, (M,), dtype=torch.int32, device=dev),
               base=torch.zeros(M, N, dtype=BF16, device=dev), dy=torch.zeros(M, N, dtype=BF16, device=dev))
    d["dy"][:20] = 0
    for k in ("x", "ids", "base", "dy"):
        big[k][held] = d[k]
    y, dx, da, db = run_all(big, AdapterRows(big["ids"], n))
    check_all(d, (y[held], dx[held], da, db))


def test_empty_batch(dev):
    d = make(0, 32, 16, 4, 2, BF16, dev)
    y, dx, da, db = run_all(d, AdapterRows(d["ids"], 2))
    assert y.shape == (0, 16) and dx.shape == (0, 32) and not da.any() and not db.any()


def test_gradients_by_differences(dev):
    """The term is linear in x, in A and in B: a difference of <y, dy> along any direction
    is the gradient's product with it, up to fp32 sums (n 2^-24 of absolute sums)."""
    d = make(50, 48, 40, 6, 2, FP32, dev, seed=11)
    rows = AdapterRows(d["ids"], 2)
    _, *grads = run_all(d, rows)
    f = lambda x, a, b: (multi_lora(x, a, b, d["s"], rows).double() * d["dy"].double()).sum()
    at = [d["x"], d["a"], d["b"]]
    for i, g in enumerate(grads):
        step = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        moved = list(at)
        moved[i] = at[i] + step
        # the step that was made, after rounding
        want = (g.double() * (moved[i].double() - at[i].double())).sum()
        big = [t.abs() for t in moved]
        s = (multi_lora(big[0], big[1], big[2], d["s"], rows).double() * d["dy"].double().abs()).sum() + \
            (multi_lora(at[0].abs(), at[1].abs(), at[2].abs(), d["s"], rows).double() * d["dy"].double().abs()).sum()
        assert abs((f(*moved) - f(*at) - want).item()) <= 4 * (48 + 40 + 50 + 6) * E32 * s.item()


def test_base_gradient_and_partial_needs(dev):
    d = make(20, 64, 48, 8, 2, BF16, dev)
    rows = AdapterRows(d["ids"], 2)
    base = d["base"].clone().requires_grad_(True)
    y = multi_lora(d["x"], d["a"], d["b"], d["s"], rows, base)
    assert torch.equal(torch.autograd.grad(y, base, d["dy"])[0], d["dy"])
    full = run_all(d, rows)[1:]
    for i, k in enumerate(("x", "a", "b")):
        t = d[k].detach().clone().requires_grad_(True)
        args = {**{q: d[q] for q in ("x", "a", "b")}, k: t}
        y = multi_lora(args["x"], args["a"], args["b"], d["s"], rows, d["base"])
        assert torch.equal(torch.autograd.grad(y, t, d["dy"])[0], full[i])


def test_broadcast_and_transposed_base(dev):
    d = make(20, 64, 48, 8, 2, BF16, dev)
    rows = AdapterRows(d["ids"], 2)
    bias = d["base"][0].clone().requires_grad_(True)
    y = multi_lora(d["x"], d["a"], d["b"], d["s"], rows, bias.expand(20, 48))
    assert torch.equal(y, multi_lora(d["x"], d["a"], d["b"], d["s"], rows, bias.detach().repeat(20, 1)))
    (db,) = torch.autograd.grad(y, bias, d["dy"])
    want = d["dy"].double().sum(0)  # torch's own sum over the broadcast rows
    assert bool(((db.double() - want).abs() <= U[BF16] * want.abs() + 20 * E32 * d["dy"].double().abs().sum(0)).all())
    turned = d["base"].t().contiguous().t()
    want = multi_lora(d["x"], d["a"], d["b"], d["s"], rows, d["base"])
    assert torch.equal(multi_lora(d["x"], d["a"], d["b"], d["s"], rows, turned), want)
    with pytest.raises(RuntimeError, match="adjacent columns"):  # in place there is no copy
        ops.multi_lora(d["x"], d["a"], d["b"], d["s"], rows.plan, turned, turned)


def test_fp32_factors_beside_16_bit_rows(dev):
    d = make(20, 64, 48, 8, 2, BF16, dev)
    rows = AdapterRows(d["ids"], 2)
    a, b = d["a"].float().requires_grad_(True), d["b"].float().requires_grad_(True)
    y = multi_lora(d["x"], a, b, d["s"], rows, d["base"])
    da, db = torch.autograd.grad(y, (a, b), d["dy"])
    want = run_all(d, rows)
    assert torch.equal(y, want[0]) and torch.equal(da, want[2].float()) and torch.equal(db, want[3].float())


def test_on_another_stream_and_in_a_graph(dev):
    d = make(100, 256, 192, 16, 4, BF16, dev)
    want = multi_lora(d["x"], d["a"], d["b"], d["s"], AdapterRows(d["ids"], 4), d["base"])
    wx = run_all(d, AdapterRows(d["ids"], 4))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = multi_lora(d["x"], d["a"], d["b"], d["s"], AdapterRows(d["ids"], 4), d["base"])
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        ids, x = d["ids"].clone(), d["x"].clone()
        with torch.cuda.graph(graph, stream=stream):
            rows = AdapterRows(ids, 4)
            y, u = ops.multi_lora(x, d["a"], d["b"], d["s"], rows.plan, d["base"], need_u=True)
            grads = ops.multi_lora_grads(x, d["dy"], d["a"], d["b"], d["s"], rows.plan, u)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for k in range(4):  # new rows and ids, read by the replays
        e = make(100, 256, 192, 16, 4, BF16, dev, seed=50 + k)
        ids.copy_(e["ids"])
        x.copy_(e["x"])
        graph.replay()
        torch.cuda.synchronize()
        eager = {**d, "x": e["x"], "ids": e["ids"]}
        for a, b in zip((y, *grads), run_all(eager, AdapterRows(e["ids"], 4))):
            assert torch.equal(a, b)
    for a, b in zip(wx, run_all(d, AdapterRows(d["ids"], 4))):
        assert torch.equal(a, b)


# ---- layers ---------------------------------------------------------------------
def quantized(K, N, bits, dev, seed=0, bias=True):
    lin = torch.nn.Linear(K, N, bias=bias)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=g) * 0.05)
    return QuantLinear.from_linear(lin.to(dev), bits=bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("M", [3, 90])
def test_layer_matches_its_parts(dev, bits, M):
    """Forward: the quantized linear's result plus the term; backward: its dX plus the
    term's, each rounded as the parts round them."""
    K, N, n, r = 128, 192, 3, 8
    d = make(M, K, N, r, n, BF16, dev, seed=bits)
    q = quantized(K, N, bits, dev)
    layer = MultiLoRALinear(q, n, r)
    with torch.no_grad():
        layer.lora_A.copy_(d["a"])
        layer.lora_B.copy_(d["b"])
        layer.scaling.copy_(d["s"])
    rows = AdapterRows(d["ids"], n)
    x = d["x"].clone().requires_grad_(True)
    y = layer(x, rows)
    y.backward(d["dy"])
    x2 = d["x"].clone().requires_grad_(True)
    base = q(x2)
    with torch.no_grad():
        assert torch.equal(y, multi_lora(d["x"], d["a"], d["b"], d["s"], rows, base))
        assert torch.equal(layer(d["x"], rows), y)
    dbase = torch.autograd.grad(base, x2, d["dy"])[0]
    dx, da, db = ops.multi_lora_grads(d["x"], d["dy"], d["a"], d["b"], d["s"], rows.plan,
                                      ops.multi_lora(d["x"], d["a"], d["b"], d["s"], rows.plan, need_u=True)[1], dx=dbase)
    assert torch.equal(x.grad, dx)
    assert torch.equal(layer.lora_A.grad, da.float()) and torch.equal(layer.lora_B.grad, db.float())


def test_attach_adapters_leaves_a_model_that_it_refuses(dev):
    def layer():
        return LoRALinear(QuantLinear.from_linear(torch.nn.Linear(64, 64).to(dev), bits=4), r=4)

    merged = torch.nn.Sequential(layer(), layer())
    merged[1].merge_lora()
    with pytest.raises(RuntimeError, match="merged"):
        attach_adapters(merged, 2)
    other = torch.nn.Sequential(layer(), layer())
    other[1].base_layer = torch.nn.Linear(64, 64).to(dev)
    with pytest.raises(TypeError, match="QuantLinear"):
        attach_adapters(other, 2)
    assert all(isinstance(m, LoRALinear) for m in (*merged, *other))
    assert not attach_adapters(torch.nn.Sequential(layer()).eval(), 2)[0].training


def test_attached_layers_cast_shared_and_without_rows(dev):
    torch.manual_seed(3)
    layer = LoRALinear(QuantLinear.from_linear(torch.nn.Linear(64, 96).to(dev), bits=4), r=4, lora_alpha=8)
    with torch.no_grad():
        layer.lora_B.normal_()
    x = torch.randn(6, 64, device=dev).to(BF16)
    want = layer(x)
    model = torch.nn.ModuleDict({"a": layer, "b": layer})  # one layer in two places
    attach_adapters(model, 2)
    assert isinstance(model["a"], MultiLoRALinear) and model["b"] is model["a"]
    alone = attach_adapters(layer, 2)  # the model is the layer
    assert isinstance(alone, MultiLoRALinear)
    alone.scaling.data = alone.scaling.data.to(BF16)  # as model.to(torch.bfloat16) leaves it
    rows = AdapterRows(torch.zeros(6, dtype=torch.int32, device=dev), 2)
    for m in (model["b"], alone):
        got = m(x, rows)
        assert ((got - want).abs() <= 2.0 ** -6 * want.abs() + 2.0 ** -6 * want.abs().max()).all()
    none = AdapterRows(torch.zeros(0, dtype=torch.int32, device=dev), 2)
    y = alone(x[:0].requires_grad_(True), none)
    y.sum().backward()
    assert y.shape == (0, 96) and not alone.lora_A.grad.any() and not alone.lora_B.grad.any()


def test_attach_adapters(dev):
    """A model of LoRALinears becomes one of many adapters: rows of adapter 0 give what the
    single-adapter layer gives (to the roundings of its intermediate, U of the term's
    absolute sum each), rows without one the base."""
    K, N, r = 128, 64, 8
    ll = LoRALinear(quantized(K, N, 4, dev), r=r)
    with torch.no_grad():
        ll.lora_B.copy_(torch.randn(N, r, generator=torch.Generator().manual_seed(1)) * 0.1)
    model = torch.nn.Sequential(torch.nn.Identity(), ll)
    x = torch.randn(30, K, generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    with torch.no_grad():
        one, base = model(x), ll.base_layer(x)
    attach_adapters(model, 4)
    assert isinstance(model[1], MultiLoRALinear) and model[1].n == 4
    with pytest.raises(RuntimeError, match="adapter rows"):
        model(x)
    ids = torch.zeros(30, dtype=torch.int32, device=dev)
    ids[10:] = -1
    assert set_adapter_rows(model, AdapterRows(ids, 4)) == 1
    with torch.no_grad():
        y = model(x)
    assert torch.equal(y[10:], base[10:])
    term = ll.scaling * (x.double().abs() @ ll.lora_A.double().abs().T @ ll.lora_B.double().abs().T)
    err = (y[:10].double() - one[:10].double()).abs()
    assert bool((err <= 2 * U[BF16] * (one[:10].double().abs() + 2 * term[:10])).all())


def test_traced_calls_are_refused_or_run_eagerly(dev):
    """torch.jit.trace raises rather than record a result that nothing fills; torch.compile
    runs the call as it is, between the traced parts."""
    d = make(12, 64, 32, 4, 2, BF16, dev)
    rows = AdapterRows(d["ids"], 2)
    f = lambda x: multi_lora(x, d["a"], d["b"], d["s"], rows, d["base"])
    with torch.no_grad():
        want = f(d["x"])
        with pytest.raises(RuntimeError):
            torch.jit.trace(f, (d["x"],), check_trace=False)
        torch._dynamo.reset()
        g = torch.compile(lambda x: f(x * 1.0) + 1.0, backend="eager")
        assert torch.equal(g(d["x"]), want + 1.0)
    x = d["x"].clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(g(x), x, d["dy"])[0], run_all(d, rows)[1])


# ---- refusals ---------------------------------------------------------------------
def test_refusals(dev):
    d = make(8, 32, 16, 4, 2, BF16, dev)
    rows = AdapterRows(d["ids"], 2)
    a, b, s = d["a"], d["b"], d["s"]
    with pytest.raises(RuntimeError, match="do not fit x"):
        multi_lora(d["x"][:7], a, b, s, rows)
    with pytest.raises(RuntimeError, match="do not fit x"):
        multi_lora(d["x"], a[:1], b[:1], s[:1], rows)
    with pytest.raises(RuntimeError, match="do not fit rows"):
        ops.multi_lora(d["x"], a[:, :, :31], b, s, rows.plan)
    with pytest.raises(TypeError, match="dtype"):
        ops.multi_lora(d["x"], a.float(), b, s, rows.plan)
    with pytest.raises(RuntimeError, match="scaling"):
        ops.multi_lora(d["x"], a, b, s[:1], rows.plan)
    with pytest.raises(RuntimeError, match="base"):
        multi_lora(d["x"], a, b, s, rows, d["base"].float())
    with pytest.raises(RuntimeError, match="rows by adapter"):
        ops.multi_lora(d["x"], a, b, s)
    with pytest.raises(RuntimeError, match="not those of"):
        ops.multi_lora(torch.cat([d["x"]] * 9), a, b, s, rows.plan)
    with pytest.raises(RuntimeError, match="u is not"):
        ops.multi_lora_grads(d["x"], d["dy"], a, b, s, rows.plan)
    with pytest.raises(RuntimeError, match="codes"):
        ops.multi_lora_grads(ops.act8_quantize(d["x"][:7]), d["dy"], a, b, s, rows.plan, need_b=False)
    with pytest.raises(RuntimeError, match="columns"):
        ops.multi_lora_grads(d["x"], d["dy"][:, :8], a, b, s, rows.plan, need_b=False)
    with pytest.raises(ValueError, match="activation_bits"):
        multi_lora(d["x"], a, b, s, rows, activation_bits=4)
    with pytest.raises(RuntimeError, match="GPU"):
        multi_lora(d["x"].cpu(), a, b, s, rows)
    with pytest.raises(RuntimeError, match="1 to 1024"):
        AdapterRows(d["ids"], 1025)
    with pytest.raises(TypeError, match="int32 or int64"):
        AdapterRows(d["ids"].float(), 2)
    with pytest.raises(RuntimeError, match="rq_multi_lora"):
        big = torch.zeros(1, 600, 32, dtype=BF16, device=dev), torch.zeros(1, 16, 600, dtype=BF16, device=dev)
        ops.multi_lora(d["x"], *big, s[:1])
    ll = LoRALinear(quantized(128, 64, 4, dev), r=16)
    with pytest.raises(ValueError, match="rank"):
        MultiLoRALinear(ll.base_layer, 2, r=8).load_adapter(0, ll)
