"""distill_loss without a GPU: its refusals, and the plain form's gradient
against differences."""

import ctypes as C

import numpy as np
import pytest
import torch

import distill_plain as P
import paged_moe_b200 as pm
from paged_moe_b200 import _lib as L


@pytest.mark.parametrize("kw,err", [
    (dict(tail="none"), ValueError), (dict(reduction="batchmean"), ValueError), (dict(temp=0.0), ValueError),
    (dict(temp=float("nan")), ValueError), (dict(temp=float("inf")), ValueError),
    (dict(logits=torch.zeros(100)), ValueError), (dict(logits=torch.zeros((3, 100), dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros((3, 0))), ValueError),
    (dict(teacher_ids=torch.zeros((2, 5), dtype=torch.int32)), ValueError),
    (dict(teacher_ids=torch.zeros((3, 5))), TypeError),
    (dict(teacher_ids=torch.zeros((3, 0), dtype=torch.int32), teacher_logprobs=torch.zeros((3, 0))), ValueError),
    (dict(teacher_logprobs=torch.zeros((3, 4))), ValueError),
    (dict(teacher_logprobs=torch.zeros((3, 5), dtype=torch.float64)), TypeError),
    (dict(weights=torch.zeros(4)), ValueError), (dict(weights=torch.zeros(3, dtype=torch.int32)), TypeError),
    (dict(), ValueError),  # host tensors
])
def test_distill_refuses(kw, err):
    a = dict(logits=torch.zeros((3, 100)), teacher_ids=torch.zeros((3, 5), dtype=torch.int32),
             teacher_logprobs=torch.zeros((3, 5)))
    a.update(kw)
    with pytest.raises(err):
        pm.distill_loss(**a)
    if a["logits"].is_floating_point():
        a["logits"] = a["logits"].requires_grad_()
        with pytest.raises(err):
            pm.distill_loss(**a)


def _d(**kw):
    d = L.Distill()
    d.logits, d.dtype, d.rows, d.vocab, d.row_stride, d.ids, d.logprobs = 0x1000, 0, 4, 1000, 1000, 0x2000, 0x3000
    d.k, d.inv_temperature, d.tail, d.reduction = 8, 1.0, 0, 2
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("bad,rc", [
    (dict(k=0), L.PM_ERR_ARG), (dict(k=257), L.PM_ERR_UNSUPPORTED), (dict(vocab=0), L.PM_ERR_ARG),
    (dict(row_stride=10), L.PM_ERR_ARG), (dict(dtype=2), L.PM_ERR_ARG), (dict(tail=2), L.PM_ERR_ARG),
    (dict(reduction=3), L.PM_ERR_ARG), (dict(inv_temperature=0.0), L.PM_ERR_ARG), (dict(ids=None), L.PM_ERR_ARG),
    (dict(logprobs=None), L.PM_ERR_ARG), (dict(logits=None), L.PM_ERR_ARG), (dict(rows=-1), L.PM_ERR_ARG),
    (dict(vocab=262145, row_stride=262145), L.PM_ERR_UNSUPPORTED),
])
def test_distill_c_checks(bad, rc):
    lib = L.load()
    assert lib.pm_distill_workspace_bytes(C.byref(_d(**bad))) == 0
    assert lib.pm_distill_loss(C.byref(_d(**bad)), 0x4000, None, 0, None, 0x5000, 1 << 20, None) == rc


def test_distill_c_outputs():
    lib = L.load()
    d = _d()
    need = lib.pm_distill_workspace_bytes(C.byref(d))
    assert lib.pm_distill_loss(C.byref(d), None, None, 0, None, 0x5000, need, None) == L.PM_ERR_ARG
    assert lib.pm_distill_loss(C.byref(d), 0x4000, 0x1000, 1000, None, 0x5000, need, None) == L.PM_ERR_ARG  # in place
    assert lib.pm_distill_loss(C.byref(d), 0x4000, 0x6000, 999, None, 0x5000, need, None) == L.PM_ERR_ARG
    assert lib.pm_distill_loss(C.byref(d), 0x4000, None, 0, None, None, need, None) == L.PM_ERR_ARG
    assert lib.pm_distill_loss(C.byref(d), 0x4000, None, 0, None, 0x5000, need - 1, None) == L.PM_ERR_WORKSPACE
    assert lib.pm_distill_scale(None, 0, 4, 1000, 1000, 0x4000, None) == L.PM_ERR_ARG
    assert lib.pm_distill_scale(0x4000, 0, 4, 1000, 999, 0x4000, None) == L.PM_ERR_ARG
    assert lib.pm_distill_scale(None, 0, 0, 1000, 1000, None, None) == L.PM_OK


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("temp", [1.0, 2.0, 0.5])
def test_plain_gradient_against_differences(tail, temp):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 30)) * 2
    ids = rng.integers(0, 30, (4, 6))
    ids[1, 3:] = -1
    ids[2, 1] = ids[2, 0]  # an id twice
    lps = np.log(rng.dirichlet(np.ones(6), 4) * 0.8)
    _, g, _ = P.rows(x, ids, lps, temp, tail)
    h = 1e-5
    for v in range(30):
        up, dn = x.copy(), x.copy()
        up[:, v] += h
        dn[:, v] -= h
        diff = (P.rows(up, ids, lps, temp, tail)[0] - P.rows(dn, ids, lps, temp, tail)[0]) / (2 * h)
        # central differences: h^2 times a third derivative of at most a few, and 1e-16 / h of rounding
        np.testing.assert_allclose(g[:, v], diff, atol=1e-8)


def test_distill_c_checks_of_alignment():
    lib = L.load()
    d = _d()
    need = lib.pm_distill_workspace_bytes(C.byref(d))
    assert lib.pm_distill_loss(C.byref(d), 0x1000, None, 0, None, 0x9008, need, None) == L.PM_ERR_ARG
    assert lib.pm_distill_loss(C.byref(d), 0x1000, 0x2002, d.vocab, None, 0x9000, need, None) == L.PM_ERR_ARG
    d = _d(logits=0x5002)
    assert lib.pm_distill_loss(C.byref(d), 0x1000, None, 0, None, 0x9000, need, None) == L.PM_ERR_ARG
    assert lib.pm_distill_scale(0x1002, 0, 1, 8, 8, 0x3000, None) == L.PM_ERR_ARG
    assert lib.pm_distill_scale(0x1000, 0, 1, 262145, 262145, 0x3000, None) == L.PM_ERR_UNSUPPORTED
