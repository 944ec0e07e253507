"""Refusals of the top-log-probability and beam entry points, before any CUDA
call (no GPU needed): Python through the extension, and the C ABI."""

import ctypes as C

import pytest
import torch

import paged_moe_b200 as pm
from paged_moe_b200 import _lib as L


def _x(B=2, W=3, V=100, dtype=torch.float32):
    return torch.zeros((B, W, V), dtype=dtype)


@pytest.mark.parametrize("kw,err", [
    (dict(k=0), ValueError), (dict(k=-3), ValueError), (dict(temp=0.0), ValueError), (dict(temp=-1.0), ValueError),
    (dict(temp=float("nan")), ValueError), (dict(temp=float("inf")), ValueError),
    (dict(logits=torch.zeros(4)), ValueError), (dict(logits=_x()), ValueError),
    (dict(logits=torch.zeros((2, 0))), ValueError),
    (dict(logits=torch.zeros((2, 100), dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros((2, 100), dtype=torch.int32)), TypeError),
    (dict(mask=torch.zeros((2, 4))), TypeError), (dict(mask=torch.zeros((2, 3), dtype=torch.int32)), ValueError),
    (dict(mask=torch.zeros((3, 4), dtype=torch.int32)), ValueError),
    (dict(), ValueError),  # host logits
])
def test_top_logprobs_refuses(kw, err):
    a = dict(logits=torch.zeros((2, 100)), k=5)
    a.update(kw)
    with pytest.raises(err):
        pm.top_logprobs(**a)


@pytest.mark.parametrize("kw,err", [
    (dict(n=0), ValueError), (dict(scores=torch.zeros(6)), ValueError),
    (dict(scores=torch.zeros((2, 3), dtype=torch.float64)), TypeError),
    (dict(scores=torch.zeros((2, 0))), ValueError),
    (dict(scores=torch.zeros((3, 2))), ValueError), (dict(logits=torch.zeros((5, 100))), ValueError),
    (dict(logits=_x(dtype=torch.float16)), TypeError),
    (dict(done=torch.zeros((2, 3), dtype=torch.bool)), ValueError),  # without eos
    (dict(done=torch.zeros((2, 3)), eos=5), TypeError),
    (dict(done=torch.zeros((2, 4), dtype=torch.bool), eos=5), ValueError),
    (dict(lengths=torch.zeros((2, 3), dtype=torch.int64)), TypeError),
    (dict(lengths=torch.zeros((6,), dtype=torch.int32)), ValueError),
    (dict(length_penalty=0.5), ValueError),  # without lengths
    (dict(length_penalty=17.0, lengths=torch.zeros((2, 3), dtype=torch.int32)), ValueError),
    (dict(length_penalty=float("nan"), lengths=torch.zeros((2, 3), dtype=torch.int32)), ValueError),
    (dict(n=4, keep_slots=True), ValueError), (dict(eos=-5), ValueError),
    (dict(mask=torch.zeros((5, 4), dtype=torch.int32)), ValueError),
    (dict(), ValueError),  # host logits
])
def test_beam_select_refuses(kw, err):
    a = dict(logits=_x(), scores=torch.zeros((2, 3)))
    a.update(kw)
    with pytest.raises(err):
        pm.beam_select(**a)


def _top(**kw):
    t = L.TopRows()
    t.logits, t.dtype, t.rows, t.vocab, t.row_stride, t.k, t.inv_temperature = 0x1000, 0, 4, 1000, 1000, 20, 1.0
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("bad,rc", [
    (dict(k=0), L.PM_ERR_ARG), (dict(k=257), L.PM_ERR_UNSUPPORTED), (dict(logits=None), L.PM_ERR_ARG),
    (dict(dtype=3), L.PM_ERR_ARG), (dict(vocab=0), L.PM_ERR_ARG), (dict(row_stride=999), L.PM_ERR_ARG),
    (dict(vocab=262145, row_stride=262145), L.PM_ERR_UNSUPPORTED), (dict(rows=-1), L.PM_ERR_ARG),
    (dict(rows=1 << 31), L.PM_ERR_UNSUPPORTED), (dict(inv_temperature=0.0), L.PM_ERR_ARG),
    (dict(inv_temperature=float("inf")), L.PM_ERR_ARG), (dict(mask=0x2000, mask_stride=31), L.PM_ERR_ARG),
])
def test_top_logprobs_c_checks(bad, rc):
    assert L.load().pm_top_logprobs(C.byref(_top(**bad)), 0x3000, 0x4000, None, None) == rc


def test_top_logprobs_c_outputs_and_empty():
    lib = L.load()
    assert lib.pm_top_logprobs(C.byref(_top()), None, 0x4000, None, None) == L.PM_ERR_ARG
    assert lib.pm_top_logprobs(None, 0x3000, 0x4000, None, None) == L.PM_ERR_ARG
    assert lib.pm_top_logprobs(C.byref(_top(rows=0)), None, None, None, None) == L.PM_OK


def _beam(**kw):
    b = L.Beam()
    b.logits, b.dtype, b.items, b.beams, b.vocab, b.row_stride = 0x1000, 0, 2, 4, 1000, 1000
    b.scores, b.eos, b.n = 0x2000, -1, 8
    for k, v in kw.items():
        setattr(b, k, v)
    return b


@pytest.mark.parametrize("bad", [
    dict(beams=0), dict(beams=65), dict(n=0), dict(n=257), dict(scores=None), dict(done=0x3000), dict(eos=-2),
    dict(length_penalty=1.0), dict(keep_slots=1), dict(vocab=0), dict(row_stride=10), dict(items=1 << 30),
    dict(length_penalty=float("nan")), dict(mask=0x5000, mask_stride=2),
])
def test_beam_select_c_checks(bad):
    lib = L.load()
    b = _beam(**bad)
    assert lib.pm_beam_select_workspace_bytes(C.byref(b)) == 0
    o = L.BeamOut()
    o.scores, o.parents, o.tokens = 0x6000, 0x7000, 0x8000
    assert lib.pm_beam_select(C.byref(b), C.byref(o), 0x9000, 1 << 30, None) in (L.PM_ERR_ARG, L.PM_ERR_UNSUPPORTED)


def test_beam_select_c_workspace_and_outputs():
    lib = L.load()
    b = _beam()
    need = lib.pm_beam_select_workspace_bytes(C.byref(b))
    assert need > 0
    o = L.BeamOut()
    o.scores, o.parents, o.tokens = 0x6000, 0x7000, 0x8000
    assert lib.pm_beam_select(C.byref(b), C.byref(o), 0x9000, need - 1, None) == L.PM_ERR_WORKSPACE
    assert lib.pm_beam_select(C.byref(b), C.byref(o), None, need, None) == L.PM_ERR_ARG
    o.tokens = None
    assert lib.pm_beam_select(C.byref(b), C.byref(o), 0x9000, need, None) == L.PM_ERR_ARG
    assert lib.pm_beam_select(C.byref(_beam(items=0)), C.byref(o), None, 0, None) == L.PM_OK
