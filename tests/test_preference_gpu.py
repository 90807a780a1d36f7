"""Preference loss and sequence log-probabilities against fp64 on the CPU.

Bounds: a row's sum of V exponentials is fp32 (V 2^-24 relative at most, of which a
tree over threads leaves far fewer; 64 + V / 2048 terms in a chain here), its
exponents differ from the row's maximum by d with d 2^-24 relative error of the
argument, that is 2^-24 |d| <= 2^-17 for |d| <= 128 in a term that is exp(-|d|) of
the sum: at most 2^-24 e^-1 |d|-weighted, under 2 2^-24.  So log-probabilities err by
(70 + V / 2048) 2^-24 each, plus the fp32 result's rounding; gradients relatively by
that and 2^-24 (2 + |z - max|), and by their dtype's rounding."""
import pytest
import torch

from rocm_qlora import ops
from rocm_qlora.losses import preference_loss, sequence_logps

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}
E32 = 2.0 ** -24
TINY = {BF16: 2.0 ** -133, FP16: 2.0 ** -24, FP32: 2.0 ** -149}


def make(lengths, V, dtype, dev, seed=0, prompt=0.3):
    g = torch.Generator().manual_seed(seed)
    T = sum(lengths)
    z = (torch.randn(T, V, generator=g) * 3).to(dtype)
    labels = torch.randint(0, V, (T,), generator=g)
    labels[torch.rand(T, generator=g) < prompt] = -100
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return z.to(dev), labels.to(dev), offsets.to(dev)


def oracle(z, labels, offsets, ref=None, beta=0.1, eps=0.0, average=False, ignore=-100, pairs=True, up=None):
    """loss, logps, dz, counts in fp64 by autograd over log_softmax."""
    z = z.detach().double().cpu().requires_grad_(True)
    labels, offsets = labels.cpu(), offsets.cpu().tolist()
    logps, counts = [], []
    for a, b in zip(offsets, offsets[1:]):
        lp, n = torch.zeros((), dtype=torch.float64), 0
        for t in range(a, b - 1):
            y = int(labels[t + 1])
            if y == ignore:
                continue
            lp = lp + torch.log_softmax(z[t], 0)[y]
            n += 1
        logps.append(lp / max(n, 1) if average else lp)
        counts.append(n)
    logps = torch.stack(logps)
    if not pairs:
        dz = torch.autograd.grad((logps * up.double().cpu()).sum(), z, allow_unused=True)[0]
        return None, logps.detach(), torch.zeros_like(z) if dz is None else dz, counts
    P = len(counts) // 2
    d = logps - (ref.double().cpu() if ref is not None else 0)
    h = beta * (d[:P] - d[P:])
    loss = -((1 - eps) * torch.nn.functional.logsigmoid(h) + eps * torch.nn.functional.logsigmoid(-h)).mean()
    dz = torch.autograd.grad(loss, z, allow_unused=True)[0] if loss.requires_grad else None
    return loss.detach(), logps.detach(), torch.zeros_like(z) if dz is None else dz, counts


def row_error(V):
    return (70 + V / 2048) * E32


def check_logps(got, want, counts, V, average):
    n = torch.tensor([1.0 if average else max(c, 1) for c in counts], dtype=torch.float64)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= n * row_error(V) + E32 * want.abs()).all()), (err, want)
    return (n * row_error(V) + E32 * want.abs())


def check_dz(got, want, z, dtype, V, extra=0.0):
    zd = z.detach().double().cpu()
    rel = row_error(V) + E32 * (4 + (zd.amax(-1, keepdim=True) - zd).clamp_max(200)) + extra
    bound = (U[dtype] + rel) * want.abs() + TINY[dtype]
    # at the target the two terms cancel: the error is of their size, |c| = sum over the others
    rows = want.abs().sum(-1, keepdim=True) / 2
    hit = want.abs() >= rows * (1 - 1e-9)
    bound = torch.where(hit, bound + rel * (2 * rows + _coef(want)), bound)
    err = (got.detach().double().cpu() - want).abs()
    worst = (err / bound).max().item()
    assert worst <= 1.0, f"dz: error {worst:.2f} times its bound"


def _coef(want):
    """|c| of a row, at most the largest over rows (rows of a sequence share it)."""
    return (want.abs().sum(-1, keepdim=True)).amax()


CASES = [
    # lengths of the sequences (an even number), V
    ([2, 2], 2),
    ([5, 3], 7),
    ([3, 4, 6, 2], 33),
    ([9, 1, 4, 12], 1000),
    ([20, 31], 5003),
    ([6, 5], 50257),
    ([40, 3, 17, 25, 8, 60], 640),
    ([3, 3], 128256),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("lengths,V", CASES)
def test_loss_and_gradient(dev, lengths, V, average, dtype):
    print(f"preference {lengths} V={V} {dtype} average={average}", flush=True)
    z, labels, offsets = make(lengths, V, dtype, dev, seed=V)
    S = len(lengths)
    ref = torch.randn(S, generator=torch.Generator().manual_seed(1)).to(dev) * 2
    z.requires_grad_(True)
    beta, eps = 0.3, 0.1
    loss, logps = preference_loss(z, labels, offsets, ref, beta=beta, label_smoothing=eps, average=average)
    dz = torch.autograd.grad(loss, z)[0]
    # what the loss is at the log-probabilities within their bounds
    wl, wp, wz, counts = oracle(z, labels, offsets, ref, beta, eps, average)
    tol = check_logps(logps, wp, counts, V, average)
    assert abs(loss.double().cpu() - wl) <= beta * tol.sum() + 2 * E32 * wl.abs()
    # the coefficient moves by beta / 4 of D's error at most, relative to one no smaller than ...
    h = beta * ((wp - ref.double().cpu())[:S // 2] - (wp - ref.double().cpu())[S // 2:])
    coef = (eps * torch.sigmoid(h) - (1 - eps) * torch.sigmoid(-h)).abs().min()
    check_dz(dz, wz, z, dtype, V, extra=float(beta * tol.sum() / 4 / coef) + 4 * E32)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_padded_batch_without_copies(dev, dtype):
    """[B, L, V] logits, contiguous or a view whose rows do not lie end to end."""
    B, L, V = 4, 11, 300
    z, labels, offsets = make([L] * B, V, dtype, dev, seed=1)
    ref = torch.zeros(B, device=dev)
    want = preference_loss(z, labels, offsets, ref)
    dense = z.view(B, L, V).clone().requires_grad_(True)
    loss, logps = preference_loss(dense, labels.view(B, L), None, ref)
    assert torch.equal(loss, want[0]) and torch.equal(logps, want[1])
    dz = torch.autograd.grad(loss, dense)[0]
    big = torch.full((B, L + 3, V + 5), float("nan"), dtype=dtype, device=dev)
    big[:, 2:2 + L, 3:3 + V] = dense.detach()
    big.requires_grad_(True)
    view = big[:, 2:2 + L, 3:3 + V]
    l2, p2 = preference_loss(view, labels.view(B, L), None, ref)
    assert torch.equal(l2, loss) and torch.equal(p2, logps)
    assert torch.equal(torch.autograd.grad(l2, big)[0][:, 2:2 + L, 3:3 + V], dz)
    l3, _ = preference_loss(view.transpose(1, 2).contiguous().transpose(1, 2), labels.view(B, L), None, ref)
    assert torch.equal(l3, loss)
    first, _, _, counts = oracle(dense.detach().view(B * L, V), labels, offsets, ref)
    assert abs(loss.item() - first.item()) <= 0.1 * 2 * sum(counts) * row_error(V) + 1e-6


@pytest.mark.parametrize("average", [False, True])
def test_sequence_logps_and_their_gradient(dev, average):
    z, labels, offsets = make([7, 1, 13, 4, 2], 130, FP32, dev, seed=2)
    up = torch.tensor([1.0, -2.0, 0.5, 0.0, 3.0], device=dev)
    z.requires_grad_(True)
    lp = sequence_logps(z, labels, offsets, average=average)
    _, wp, wz, counts = oracle(z, labels, offsets, average=average, pairs=False, up=up)
    check_logps(lp, wp, counts, 130, average)
    check_dz(torch.autograd.grad(lp, z, up)[0], wz, z, FP32, 130, extra=4 * E32)
    with torch.no_grad():
        assert torch.equal(sequence_logps(z, labels, offsets, average=average), lp)


def test_gradient_by_differences(dev):
    """Central differences of the loss along random directions.  With step h the
    difference errs by h^2 / 6 of a third derivative (under 1 here) and by the loss's
    rounding, 2^-23 loss / h."""
    z, labels, offsets = make([9, 6, 7, 12], 40, FP32, dev, seed=3)
    ref = torch.tensor([-20.0, -10.0, -15.0, -30.0], device=dev)
    z.requires_grad_(True)
    f = lambda t: preference_loss(t, labels, offsets, ref, beta=0.05, label_smoothing=0.1)[0]
    loss = f(z)
    dz = torch.autograd.grad(loss, z)[0].double()
    for k in range(4):
        v = torch.randn(z.shape, generator=torch.Generator().manual_seed(k)).to(dev)
        v /= v.norm()
        h = 2.0 ** -4
        a, b = (z + h * v).detach(), (z - h * v).detach()
        want = (dz * (a.double() - b.double())).sum()
        got = f(a).double() - f(b).double()
        assert abs((got - want).item()) <= h ** 3 / 3 + 8 * E32 * (1 + loss.item()) + 34 * 0.05 * row_error(40)


def test_upstream_gradient_scales(dev):
    z, labels, offsets = make([6, 5], 64, FP32, dev)
    z.requires_grad_(True)
    one = torch.autograd.grad(preference_loss(z, labels, offsets)[0], z)[0]
    four = torch.autograd.grad(4 * preference_loss(z, labels, offsets)[0], z)[0]
    assert torch.equal(four, 4 * one)  # a power of two: exact


def test_sequences_that_do_not_count(dev):
    """Sequences of no token, of one token, without labels: log-probability 0, no gradient."""
    z, labels, _ = make([12], 50, FP32, dev, prompt=0.0)
    offsets = torch.tensor([0, 0, 1, 6, 12], dtype=torch.int32, device=dev)  # empty, one token, five, six
    labels[1:6] = -100
    z.requires_grad_(True)
    for average in (False, True):
        loss, logps = preference_loss(z, labels, offsets, average=average)
        wl, wp, wz, counts = oracle(z, labels, offsets, average=average)
        assert counts == [0, 0, 0, 5] and not logps[:3].any()
        check_logps(logps, wp, counts, 50, average)
        dz = torch.autograd.grad(loss, z)[0]
        assert not dz[:6].any() and not dz[11].any()
        check_dz(dz, wz, z, FP32, 50, extra=5 * row_error(50))
    # rows outside of every sequence
    inner = torch.tensor([2, 5, 9], dtype=torch.int64, device=dev)
    dz = torch.autograd.grad(preference_loss(z, labels.clamp_min(0), inner)[0], z)[0]
    assert not dz[:2].any() and not dz[4].any() and not dz[8:].any() and bool(dz[2:4].any())
    # nothing counts at all
    loss, logps = preference_loss(z, torch.full_like(labels, -100), offsets)
    assert not logps.any() and abs(loss.item() - 0.6931471805599453) < 1e-7
    assert not torch.autograd.grad(loss, z)[0].any()


@pytest.mark.parametrize("V", [9, 3000])
def test_masked_logits(dev, V):
    """-inf logits, rows of the type's lowest value, infinities and NaN: what log_softmax gives."""
    z, labels, offsets = make([8, 8, 8, 8], V, FP32, dev, prompt=0.0)
    z[0, : V // 2] = float("-inf")
    labels[1] = V - 1
    z[1] = torch.finfo(FP32).min
    z[2, 1:] = float("-inf")
    labels[3] = 0                       # the one token that is left
    z.requires_grad_(True)
    loss, logps = preference_loss(z, labels, offsets)
    _, wp, wz, counts = oracle(z, labels, offsets)
    check_logps(logps, wp, counts, V, False)
    dz = torch.autograd.grad(loss, z)[0]
    assert not dz[0, : V // 2].any() and bool(torch.isfinite(dz).all())
    assert torch.equal(dz[2], torch.zeros_like(dz[2]))
    z = z.detach().clone()
    z[9, 2], z[17, 1], z[25] = float("nan"), float("inf"), float("-inf")
    got = sequence_logps(z, labels, offsets)
    assert bool(torch.isfinite(got[0])) and bool(got[1:].isnan().all())
    z[10:16, :] = 0.0
    z[9] = 0.0
    z[9, int(labels[10])] = float("-inf")  # the label itself is masked
    got = sequence_logps(z, labels, offsets)
    assert got[1].item() == float("-inf")


def test_labels_outside_the_vocabulary(dev):
    """No read out of range: the sequence is NaN, the others are not touched; ignore_index may be any value."""
    z, labels, offsets = make([6, 6, 6, 6], 33, FP32, dev, prompt=0.0)
    labels[3], labels[8] = 33, -5
    want = sequence_logps(z, labels.clamp(0, 32), offsets)
    got = sequence_logps(z, labels, offsets)
    assert bool(got[:2].isnan().all()) and torch.equal(got[2:], want[2:])
    z.requires_grad_(True)
    dz = torch.autograd.grad(sequence_logps(z, labels, offsets), z, torch.ones(4, device=dev))[0]
    assert bool(dz[2].isnan().all()) and bool(dz[7].isnan().all()) and bool(torch.isfinite(dz[[0, 1, 3, 6, 12, 18]]).all())
    skip = sequence_logps(z, labels, offsets, ignore_index=33)
    assert bool(torch.isfinite(skip[0])) and bool(skip[1].isnan())


def test_offsets_that_are_no_sequences(dev):
    """Offsets past the rows or not ascending read nothing out of range."""
    z, labels, _ = make([10], 16, FP32, dev, prompt=0.0)
    for offsets in ([0, 5, 4000], [-7, 3, 10], [9, 2, 6], [0, 2 ** 30, 10]):
        got = sequence_logps(z, labels, torch.tensor(offsets, device=dev))
        assert got.shape == (2,)


def test_more_than_2_to_the_31_logits(dev):
    T, V = 70000, 32000
    z = torch.zeros(T, V, dtype=BF16, device=dev)
    g = torch.Generator().manual_seed(0)
    z[-8:] = torch.randn(8, V, generator=g).to(BF16).to(dev)
    labels = torch.full((T,), -100, device=dev)
    labels[-4:] = torch.tensor([5, 31999, 0, 77], device=dev)
    offsets = torch.tensor([0, 8, T], device=dev)
    z.requires_grad_(True)
    lp = sequence_logps(z, labels, offsets)
    want = torch.log_softmax(z[-5:-1].detach().double(), 1)[torch.arange(4), labels[-4:]].sum().item()
    assert lp[0].item() == 0.0 and abs(lp[1].item() - want) <= 4 * row_error(V) + E32 * abs(want)
    dz = torch.autograd.grad(lp, z, torch.ones(2, device=dev))[0]
    p = -torch.softmax(z[-5:-1].detach().double(), 1)
    p[torch.arange(4), labels[-4:]] += 1
    assert bool(((dz[-5:-1].double() - p).abs() <= 2.0 ** -8 * p.abs() * 1.01).all())
    assert not dz[-1].any() and not dz[:100].any() and not dz[T - 200:T - 5].any()


def test_repeats_exactly_on_other_streams_and_in_a_graph(dev):
    z, labels, offsets = make([30, 12, 25, 40], 3000, BF16, dev)
    ref = torch.randn(4, device=dev)
    want = preference_loss(z, labels, offsets, ref)
    wz = ops.preference_backward(z, ops.preference_forward(z, labels, offsets, ref)[2], torch.ones((), device=dev))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    one = torch.ones((), device=dev)
    graph = torch.cuda.CUDAGraph()
    zz = z.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = preference_loss(z, labels, offsets, ref)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            loss, logps, state = ops.preference_forward(zz, labels, offsets, ref)
            dz = ops.preference_backward(zz, state, one)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for k in range(4):
        zz.copy_(z.roll(k, 1))
        graph.replay()
        torch.cuda.synchronize()
        e = ops.preference_forward(z.roll(k, 1), labels, offsets, ref)
        assert torch.equal(loss, e[0]) and torch.equal(logps, e[1])
        assert torch.equal(dz, ops.preference_backward(z.roll(k, 1), e[2], one))
        if k == 0:
            assert torch.equal(dz, wz)


def test_refusals(dev):
    z, labels, offsets = make([4, 4], 16, FP32, dev)
    with pytest.raises(RuntimeError, match="offsets"):
        preference_loss(z, labels)
    with pytest.raises(RuntimeError, match="offsets"):
        preference_loss(z, labels, offsets.float())
    with pytest.raises(RuntimeError, match="packed"):
        preference_loss(z.view(2, 4, 16), labels.view(2, 4), offsets)
    with pytest.raises(RuntimeError, match="no pairs"):
        preference_loss(z, labels, offsets[:2])
    with pytest.raises(RuntimeError, match="labels"):
        preference_loss(z, labels.int(), offsets)
    with pytest.raises(RuntimeError, match="labels"):
        preference_loss(z, labels[:7], offsets)
    with pytest.raises(RuntimeError, match="ref_logps"):
        preference_loss(z, labels, offsets, torch.zeros(3, device=dev))
    with pytest.raises(ValueError, match="label_smoothing"):
        preference_loss(z, labels, offsets, label_smoothing=1.5)
    with pytest.raises(RuntimeError, match="GPU"):
        preference_loss(z.cpu(), labels, offsets)
    with pytest.raises(TypeError, match="dtype"):
        preference_loss(z.double(), labels, offsets)
    with pytest.raises(RuntimeError, match="a row at least"):
        preference_loss(z[:0], labels[:0], offsets)
