"""What the MXFP4 linears' autograd function keeps for the backward pass, with the kernels replaced by torch on the CPU."""
import pytest
import torch

from rocm_qlora import ExpertRows, MXFP4Linear, MXFP4Tensor, mxfp4_expert_linear, mxfp4_linear, ops


@pytest.fixture
def no_kernels(monkeypatch):
    def forward(x, codes, scales, K, bias, bits, plan, M):
        return x.new_ones(x.shape[0] if M is None else M, codes.shape[-2])

    def dx(dy, codes, scales, K, E, N, plan, shared):
        return dy.new_full((dy.shape[0] // shared, K), float(codes.flatten()[0]))

    monkeypatch.setattr(ops, "_mx4_linear", forward)
    monkeypatch.setattr(ops, "_mx4_dx", dx)


def held(*lead):
    return MXFP4Tensor(torch.ones(*lead, 64, dtype=torch.uint8), torch.ones(*lead, 4, dtype=torch.uint8), 100)


def expert_rows(T, k, n):
    rows = ExpertRows.__new__(ExpertRows)
    rows.M, rows.n, rows.k, rows.plan = T * k, n, k, None
    return rows


def test_a_weight_changed_between_forward_and_backward_is_refused(no_kernels):
    """As autograd refuses it for the tensors that it saves (load_state_dict writes in place)."""
    x = torch.ones(6, 100, requires_grad=True)
    w = held(16)
    for change in (lambda w: w.codes.zero_(), lambda w: w.scales.add_(1), lambda w: w.codes[3, :2].fill_(7)):
        y = mxfp4_linear(x, w)
        change(w)
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()
    we = held(3, 16)
    y = mxfp4_expert_linear(x, we, expert_rows(6, 2, 3))
    we.codes[1].zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    m = MXFP4Linear(100, 16, bias=False)
    y = m(x)
    m.load_state_dict(MXFP4Linear(100, 16, bias=False).state_dict())
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    # another forward pass sees the new weight, and has its gradient
    (dx,) = torch.autograd.grad(m(x).sum(), x)
    assert bool((dx == 0).all())


def test_a_weight_that_stays_is_taken_however_it_was_made(no_kernels):
    x = torch.ones(6, 100, requires_grad=True)
    with torch.inference_mode():
        made = held(16)
    for w in (held(16), made):
        y = mxfp4_linear(x, w)
        for _ in range(2):
            (dx,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
            assert bool((dx == 1).all())
