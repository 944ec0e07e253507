"""Temperatures whose inverse fp32 exponents cannot hold are refused, by the
Python layer and by the C ABI (no GPU needed)."""

import ctypes as C

import pytest
import torch

import paged_moe_b200 as pm
from paged_moe_b200 import _lib as L

_LOG2E = 1.4426950408889634


@pytest.mark.parametrize("temp,fits", [(1e-300, False), (1e-40, False), (4.2e-39, False), (4.3e-39, True), (1.0, True),
                                       (2e45, True), (2.1e45, False), (1e300, False)])
def test_python(temp, fits):
    match = "CUDA" if fits else "temp"
    with pytest.raises(ValueError, match=match):
        pm.top_logprobs(torch.zeros((2, 100)), 5, temp=temp)
    with pytest.raises(ValueError, match=match):
        pm.distill_loss(torch.zeros((3, 100)), torch.zeros((3, 5), dtype=torch.int32), torch.zeros((3, 5)), temp=temp)


@pytest.mark.parametrize("inv,fits", [
    (2.0 ** 128 / _LOG2E, False),             # rounds to infinity
    (2.0 ** 128 * (1 - 2.0 ** -24) / _LOG2E, True),
    (1.0, True), (2.0 ** -149 / _LOG2E, True),
    (2.0 ** -150.5 / _LOG2E, False),          # rounds to 0
    (0.0, False), (-1.0, False), (float("nan"), False), (float("inf"), False)])
def test_c(inv, fits):
    lib = L.load()
    d = L.Distill()
    d.logits, d.dtype, d.rows, d.vocab, d.row_stride, d.ids, d.logprobs = 0x1000, 0, 4, 1000, 1000, 0x2000, 0x3000
    d.k, d.inv_temperature, d.tail, d.reduction = 8, inv, 0, 2
    assert (lib.pm_distill_workspace_bytes(C.byref(d)) > 0) == fits
    t = L.TopRows()
    t.logits, t.dtype, t.rows, t.vocab, t.row_stride, t.k, t.inv_temperature = 0x1000, 0, 0, 1000, 1000, 20, inv
    assert lib.pm_top_logprobs(C.byref(t), None, None, None, None) == (L.PM_OK if fits else L.PM_ERR_ARG)
