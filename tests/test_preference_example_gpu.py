"""The example runs the new operators together: both users' adapters learn their own
preference in one batch, rows without an adapter stay the reference model."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "preference_tuning.py"
    spec = importlib.util.spec_from_file_location("preference_tuning", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_two_users_learn_in_one_batch(dev, example):
    users = 2
    model = example.build(users, dev)
    tokens, labels, user = example.pairs(users, 6, 33, dev)
    losses, reference = example.train(model, users, tokens, labels, user, 6, log=lambda *_: None)
    # before the first step the policy is the reference: every log ratio is 0
    assert abs(losses[0].item() - 0.6931472) < 1e-5
    assert losses[-1] < 0.8 * losses[0]
    # every user's pairs are told apart by its own adapter: the loss's log ratios are positive on average
    L, P = tokens.shape[1], len(user) // 2
    example.set_adapter_rows(model, example.adapter_rows(user, L, users))
    with torch.no_grad():
        ratio = example.sequence_logps(model(tokens), labels) - reference
    for u in range(users):
        assert (ratio[:P] - ratio[P:])[user[:P] == u].mean() > 0
    # without adapters nothing changed, in a batch of its own and beside rows that have one
    example.set_adapter_rows(model, example.adapter_rows(torch.full_like(user, -1), L, users))
    with torch.no_grad():
        assert torch.equal(example.sequence_logps(model(tokens), labels), reference)
    prompts, asked = tokens[[0, 6, 0, 6], :11], torch.tensor([0, 1, -1, -1], dtype=torch.int32, device=dev)
    mixed = example.answer(model, users, prompts, asked)
    none = example.answer(model, users, prompts, torch.full_like(asked, -1))
    assert torch.equal(mixed[2:], none[2:]) and not torch.equal(mixed[:2], none[:2])


def test_frozen_adapter_beside_a_trained_one(dev, example):
    """Only rows of adapter 0 have a loss: adapter 1 gets no gradient at all."""
    model = example.build(2, dev)
    tokens, labels, user = example.pairs(2, 2, 17, dev)
    example.set_adapter_rows(model, example.adapter_rows(user, 17, 2))
    only0 = torch.where((user == 0)[:, None], labels, torch.full_like(labels, example.IGNORE))
    example.preference_loss(model(tokens), only0)[0].backward()
    for m in model.modules():
        if hasattr(m, "lora_B"):
            assert not m.lora_B.grad[1].any() and bool(m.lora_B.grad[0].any())
