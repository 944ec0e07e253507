"""top_logprobs and distill_loss at the smallest and largest temperatures that
they take.  Tolerances are those of the ordinary ones: only distances from a
row's largest logit, in temperatures, enter them."""

import numpy as np
import pytest
import torch

import beam_plain as P
import distill_plain as D
import paged_moe_b200 as pm
from test_gpu_beam import _close, _logits
from test_gpu_distill import DEV, _case, _check_grad, _check_loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temp", [4.3e-39, 1e-38, 1e-30, 1e30, 1e45, 2e45])
@pytest.mark.parametrize("V", [300, 20011])
def test_top_logprobs(V, temp, dtype):
    x = _logits(1, 6, V, dtype)
    x[0] = 0.0
    x[1] = -3.0
    x[2, 1:] = float("-inf")
    x[3, 5] = x[3].max()  # two largest
    got = pm.top_logprobs(x, 7, temp=temp)
    ids, lp, _ = P.top_logprobs(x.double().cpu().numpy(), 7, temp)
    np.testing.assert_array_equal(got["ids"].cpu().numpy(), ids)
    # what fp32 cannot hold is infinite, as a log-probability of nothing is
    _close(got["logprobs"], np.where(lp <= -2.0 ** 128 * (1 - 2.0 ** -25), -np.inf, lp))


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temp", [1e-36, 1e-20, 1e20, 1e30])
@pytest.mark.parametrize("N,V", [(3, 20011), (400, 900)])
def test_distill_loss(N, V, temp, dtype, tail):
    x, ids, lps = _case(2, N, V, 6, dtype, temp=temp)
    x[1] = 0.0
    leaf = x.detach().requires_grad_()
    loss = pm.distill_loss(leaf, ids, lps, temp=temp, tail=tail, reduction="none")
    want, grad, sizes = D.loss(x.double().cpu().numpy(), ids.cpu().numpy(), lps.double().cpu().numpy(), temp, tail, None,
                               "none")
    _check_loss(loss, want)
    _check_grad(torch.autograd.grad(loss.sum(), leaf)[0], grad, sizes)


def test_what_is_refused_beside_them():
    """4.2e-39 gave ids -1 and NaN for rows with a zero, 1e300 log-probabilities
    off by 128 log 2 for rows with a -inf or of an uneven length."""
    x, ids, lps = _case(3, 2, 50, 3)
    for temp in (4.2e-39, 2.1e45, 1e300):
        with pytest.raises(ValueError, match="temp"):
            pm.top_logprobs(x, 3, temp=temp)
        with pytest.raises(ValueError, match="temp"):
            pm.distill_loss(x, ids, lps, temp=temp)
