"""distill_loss where one CTA takes several rows after one another: rings that
go on from row to row, marks handed on, and rows that are read differently or
not at all between ordinary ones.  Tolerances are those of test_gpu_distill.

There are two CTAs an SM, so that of 1,000 rows most take four or three.  The
61 base rows come round in another order for every CTA.
"""

import numpy as np
import pytest
import torch

import distill_plain as P
import paged_moe_b200 as pm
from test_gpu_distill import DEV, _case, _check_grad, _check_loss

pytestmark = pytest.mark.gpu
BASE, ROWS, K = 61, 1000, 9


def _inputs(V, dtype, pad):
    base, ids, lps = _case(90, BASE, V, K, dtype)
    lps = torch.log_softmax(lps, 1) - 0.2
    base[3] *= 3.0e6  # far from zero: summed once more from its largest
    base[4] = torch.finfo(dtype).min
    ids[9] = -1  # no entries
    base[14] = float("-inf")
    base[14, [0, V // 2, V - 1]] = torch.tensor([1.0, 2.0, 0.5], dtype=dtype, device=DEV)
    ids[14, :3] = torch.tensor([V - 1, 0, V // 2], dtype=torch.int32, device=DEV)
    ids[14, 3:] = -1
    base[20, V // 3] = float("nan")
    base[27] *= -3.0e6
    ids[28] = -1
    base[28] *= 3.0e6  # both at once
    ids[35, 2:] = V
    ids[41] = torch.arange(K, dtype=torch.int32, device=DEV)  # marks at the row's beginning
    ids[42] = torch.arange(V - K, V, dtype=torch.int32, device=DEV)  # and at its end
    base[50] = 1.0
    order = torch.arange(ROWS, device=DEV) % BASE
    store = torch.zeros(ROWS * (V + pad) + 1, dtype=dtype, device=DEV)
    x = store[1:].view(ROWS, V + pad)[:, :V]
    x.copy_(base[order])
    w = np.random.default_rng(91).random(ROWS).astype(np.float32) + 0.25
    w[150:158] = 0.0
    w[7::13] = 0.0
    w[ROWS - 3:] = 0.0
    return base, ids, lps, order, x, w


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype,V,pad,train", [(torch.float32, 9001, 2, True), (torch.bfloat16, 20011, 3, True),
                                               (torch.float32, 17003, 1, False), (torch.bfloat16, 33005, 5, False)])
def test_many_rows_of_a_cta(dtype, V, pad, train, tail):
    base, ids, lps, order, x, w = _inputs(V, dtype, pad)
    with np.errstate(invalid="ignore"):
        losses, grads, sizes = P.rows(base.double().cpu().numpy(), ids.cpu().numpy(), lps.double().cpu().numpy(), 1.0, tail)
    at = order.cpu().numpy()
    weights = torch.from_numpy(w).to(DEV)
    on = w != 0
    losses, w64 = np.where(on, losses[at], 0.0), w.astype(np.float64)
    bad = np.isnan(losses)
    assert bad.sum() >= 10
    leaf = x.detach().requires_grad_(train)
    loss = pm.distill_loss(leaf, ids[order], lps[order], tail=tail, weights=weights, reduction="none")
    got = loss.detach().double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), bad)
    # a loss is within its tolerance before its weight is applied; at 1.25 or less, after it too
    tol = 1.25 * (2 * 1.1e-5 + np.abs(losses) * 2.0 ** -23)
    assert (np.abs(got - losses * w64) <= tol)[~bad].all()
    if not train:
        return
    (grad,) = torch.autograd.grad(loss.sum(), leaf)
    for i in range(ROWS):
        if not on[i]:
            assert not grad[i].any(), i
        elif bad[i]:
            assert torch.isnan(grad[i]).all(), i
        else:
            b = at[i]
            _check_grad(grad[i], grads[b] * w64[i], sizes[b] * w64[i])


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype,V", [(torch.float32, 9001), (torch.bfloat16, 20011)])
def test_many_rows_of_a_cta_as_one_loss(dtype, V, tail):
    base, ids, lps, order, x, w = _inputs(V, dtype, 0)
    weights = torch.from_numpy(w).to(DEV)
    weights[order == 20] = 0.0  # the row without a distribution
    w = weights.cpu().numpy()
    with np.errstate(invalid="ignore"):
        losses, grads, sizes = P.rows(base.double().cpu().numpy(), ids.cpu().numpy(), lps.double().cpu().numpy(), 1.0, tail)
    at, share = order.cpu().numpy(), w.astype(np.float64) / w.astype(np.float64).sum()
    leaf = x.detach().requires_grad_()
    loss = pm.distill_loss(leaf, ids[order], lps[order], tail=tail, weights=weights)
    _check_loss(loss, np.where(w != 0, losses[at], 0.0) @ share)
    (grad,) = torch.autograd.grad(loss, leaf)
    for i in range(ROWS):
        if w[i] == 0:
            assert not grad[i].any(), i
        else:
            _check_grad(grad[i], grads[at[i]] * share[i], sizes[at[i]] * share[i])
