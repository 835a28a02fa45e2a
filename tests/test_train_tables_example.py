"""The example that trains a token table, layer norms and a vocabulary projection
with the framework's operators: its loss starts at that of a guess and falls."""

import importlib.util
import math
from pathlib import Path

import pytest
import torch

GPU = pytest.param("cuda", marks=pytest.mark.gpu)


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "train_tables.py"
    spec = importlib.util.spec_from_file_location("train_tables", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("vocab,hidden", [(300, 64), (1001, 72)])
def test_loss_falls(device, vocab, hidden):
    lines = []
    losses = _example().train(steps=30, vocab=vocab, hidden=hidden, device=device, log=lines.append)
    # logits of the untrained head have a standard deviation of a half: the loss of a guess and some 0.13
    assert abs(losses[0] - math.log(vocab)) < 0.5
    assert losses[-1] < 0.25 * losses[0] and len(lines) == 4


@pytest.mark.gpu
def test_first_loss_and_gradients_match_fp32_on_the_cpu():
    ex = _example()
    ids, targets = ex.batch(300, 8, 32, 299, torch.Generator().manual_seed(3))
    both = []
    for device, dtype in (("cuda", torch.bfloat16), ("cpu", torch.float32)):
        model = ex.SuccessorModel(300, 64, torch.device(device), torch.bfloat16, seed=0)
        with torch.no_grad():
            for t in model.tensors:
                t.data = t.data.to(dtype)
        loss = model.loss(ids.to(device), targets.to(device))
        both.append((float(loss.detach()), [g.double().cpu() for g in torch.autograd.grad(loss, model.tensors)]))
    (a, ga), (b, gb) = both
    assert abs(a - b) < 0.02 * b
    # bf16 activations through the whole model: a few rounding steps of 2^-8 each
    for x, y in zip(ga, gb):
        assert float((x - y).norm()) < 0.04 * float(y.norm())
