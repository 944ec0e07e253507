"""distill_loss with an id listed twice: two outcomes of the teacher in the
loss, their sum in the gradient.  Tolerances as in test_gpu_distill."""

import numpy as np
import pytest
import torch

import paged_moe_b200 as pm
from test_gpu_distill import DEV, REL

pytestmark = pytest.mark.gpu


def _run(x, ids, p, tail):
    leaf = x.detach().requires_grad_()
    lps = torch.log(torch.tensor([p], device=DEV))
    loss = pm.distill_loss(leaf, torch.tensor([ids], device=DEV, dtype=torch.int32), lps, tail=tail, reduction="none")
    return float(loss.detach()), torch.autograd.grad(loss.sum(), leaf)[0]


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_an_id_twice_differs_from_its_sum_by_a_constant(tail):
    x = torch.from_numpy(np.random.default_rng(1).standard_normal((1, 500)).astype(np.float32)).to(DEV)
    twice, g2 = _run(x, [7, 40, 7, 7], [0.2, 0.1, 0.3, 0.05], tail)
    once, g1 = _run(x, [7, 40], [0.55, 0.1], tail)
    # 0.55 and 0.65 of float32 probabilities; under "drop" divided by their sum
    by = 0.65 if tail == "drop" else 1.0
    apart = sum(p / by * np.log(p / 0.55) for p in (0.2, 0.3, 0.05))
    # both losses are off by 2 REL, and logarithms that float32 rounds by 2.4 * 2^-24 a unit of mass
    assert abs(twice - once - apart) <= 4 * REL + 4 * 3.0 * 2.0 ** -24
    # q is the same; probabilities move by the same roundings
    assert (g2 - g1).abs().max() <= 4 * 3.0 * 2.0 ** -24


def test_a_certain_student_of_a_token_listed_twice():
    """The divergence of the sum is 0, that of the two halves log 1/2."""
    x = torch.full((1, 300), -500.0, device=DEV)
    x[0, 9] = 500.0
    loss, grad = _run(x, [9, 9], [0.5, 0.5], "drop")
    assert abs(loss - np.log(0.5)) <= 2 * REL and not grad.abs().max() > 2.0 ** -22
