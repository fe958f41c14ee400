"""The example model: whole sequences, chunks of them and single tokens have to agree, and training has to learn."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parent.parent / "examples" / "retention_layer.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("retention_layer", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture()
def model(example):
    torch.manual_seed(1)
    return example.RetentionModel(width=128, layers=2, heads=4, key_heads=2, head_dim=32).cuda()


def near(a, b):
    # fp32 all through (matrix products in full fp32): two layers of sums of at most a few hundred terms, 2^-24 each, with room
    return ((a - b).norm() / b.norm()).item() <= 1e-4


def test_prompt_in_parts_and_single_tokens_continue_each_other(model):
    tokens = torch.randint(0, 512, (3, 60), device="cuda")
    with torch.no_grad():
        whole, last = model(tokens, keep_states=True)
        head, states = model(tokens[:, :37], keep_states=True)
        tail, states = model(tokens[:, 37:50], states=states, first=37, keep_states=True)
        assert near(torch.cat([head, tail], 1), whole[:, :50])
        pool = [torch.zeros(7, *s.shape[1:], device="cuda") for s in states]      # the sequences' states lie in a pool
        slots = torch.tensor([5, 0, 3], device="cuda", dtype=torch.int32)
        for p, s in zip(pool, states):
            p[slots.long()] = s
        for t in range(50, 60):
            step = model.step(tokens[:, t], torch.full((3,), t, device="cuda"), pool, slots)
            assert near(step, whole[:, t])
        for p, s in zip(pool, last):
            assert near(p[slots.long()], s)


def test_documents_in_a_row_do_not_see_each_other(model):
    tokens = torch.randint(0, 512, (2, 80), device="cuda")
    starts = torch.zeros(2, 80, dtype=torch.bool, device="cuda")
    starts[:, [0, 33]] = True
    with torch.no_grad():
        both = model(tokens, starts=starts)
        second = model(tokens[:, 33:], first=33)
    assert near(both[:, 33:], second)


def test_ragged_prompts(model):
    tokens = torch.randint(0, 512, (3, 50), device="cuda")
    lengths = torch.tensor([50, 21, 1], device="cuda", dtype=torch.int32)
    with torch.no_grad():
        logits, states = model(tokens, lengths=lengths, keep_states=True)
        for i, n in enumerate(lengths.tolist()):
            alone, own = model(tokens[i:i + 1, :n], keep_states=True)
            assert near(logits[i, :n], alone[0])
            assert all(near(s[i], o[0]) for s, o in zip(states, own))


def test_training_learns(example):
    torch.manual_seed(2)
    model = example.RetentionModel(width=128, layers=2, heads=4, key_heads=2, head_dim=32).cuda()
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(40):
        tokens = (torch.randint(0, 512, (8, 1), device="cuda") + torch.arange(65, device="cuda")) % 512
        loss = torch.nn.functional.cross_entropy(model(tokens[:, :-1]).flatten(0, 1), tokens[:, 1:].flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert losses[-1] < 0.7 * losses[0]
