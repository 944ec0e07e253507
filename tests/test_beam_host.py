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


_PAR = torch.zeros((2, 3), dtype=torch.int32)


@pytest.mark.parametrize("states,kw,err", [
    (torch.zeros(5, 4), {}, ValueError),                               # rows
    (torch.zeros(6, 4), dict(parents=_PAR.long()), TypeError),
    (torch.zeros(6, 4), dict(parents=_PAR[0]), ValueError),
    (torch.zeros(6, 4), dict(seq_dim=1), ValueError),                  # without lengths
    (torch.zeros(6, 4), dict(seq_dim=0, lengths=_PAR), ValueError),
    (torch.zeros(6, 4), dict(seq_dim=2, lengths=_PAR), ValueError),
    (torch.zeros(6, 4), dict(seq_dim=-3, lengths=_PAR), ValueError),
    (torch.zeros(6, 4), dict(seq_dim=[1, 1], lengths=_PAR), ValueError),
    (torch.zeros(6, 4), dict(lengths=_PAR.long()), TypeError),
    (torch.zeros(6, 4), dict(lengths=_PAR[:, :2]), ValueError),
    (torch.zeros(1, 4).expand(6, 4), {}, ValueError),                  # rows that share memory
    (torch.zeros(6, 4, 1).expand(6, 4, 5), {}, ValueError),
    (torch.zeros(6, 4, 5, 7).permute(0, 3, 1, 2)[:, :, ::2], {}, ValueError),  # does not collapse
    (torch.zeros(6, 5, 4).transpose(1, 2), dict(seq_dim=1, lengths=_PAR), ValueError),  # not dense behind dim 1
    (torch.zeros(6, 4), dict(out=torch.zeros(6, 5)), ValueError),
    (torch.zeros(6, 4), dict(out=torch.zeros(6, 4, dtype=torch.int32)), ValueError),
    (torch.zeros(6, 4), dict(out=[]), ValueError),
    (torch.zeros(6, 4), {}, ValueError),                               # host tensors
])
def test_beam_reorder_refuses(states, kw, err):
    a = dict(parents=_PAR)
    a.update(kw)
    with pytest.raises(err):
        pm.beam_reorder(states, **a)


def test_beam_reorder_refuses_the_same_memory_twice():
    t, u = torch.zeros(6, 4), torch.zeros(6, 4)
    with pytest.raises(ValueError, match="share"):
        pm.beam_reorder([t, t], _PAR)
    with pytest.raises(ValueError, match="share"):
        pm.beam_reorder([t, u], _PAR, out=[u, torch.zeros(6, 4)])
    with pytest.raises(ValueError, match="share"):
        pm.beam_reorder(t, _PAR, out=t)


def _state(**kw):
    s = L.State()
    s.src = s.dst = 0x10000
    s.src_row_stride = s.dst_row_stride = 256
    s.outer, s.run_bytes = 1, 256
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("bad,call,rc", [
    (dict(outer=0), {}, L.PM_ERR_ARG), (dict(run_bytes=-1), {}, L.PM_ERR_ARG), (dict(src=None), {}, L.PM_ERR_ARG),
    (dict(pos_bytes=100), {}, L.PM_ERR_ARG), (dict(dst_row_stride=512), {}, L.PM_ERR_ARG),
    ({}, dict(beams=0), L.PM_ERR_ARG), ({}, dict(beams=65, stride=65), L.PM_ERR_UNSUPPORTED),
    ({}, dict(parents=None), L.PM_ERR_ARG), ({}, dict(stride=1), L.PM_ERR_ARG), ({}, dict(items=-1), L.PM_ERR_ARG),
    ({}, dict(n=129), L.PM_ERR_UNSUPPORTED), ({}, dict(n=-1), L.PM_ERR_ARG),
])
def test_beam_reorder_c_checks(bad, call, rc):
    a = dict(n=1, parents=0x2000, stride=4, items=2, beams=4)
    a.update(call)
    arr = (L.State * max(1, a["n"]))(*[_state(**bad) for _ in range(max(1, a["n"]))])
    got = L.load().pm_beam_reorder(arr, a["n"], a["parents"], a["stride"], None, a["items"], a["beams"], None)
    assert got == rc


def test_beam_reorder_c_nothing_to_do():
    arr = (L.State * 1)(_state(run_bytes=0))
    lib = L.load()
    assert lib.pm_beam_reorder(arr, 1, 0x2000, 4, None, 2, 4, None) == L.PM_OK
    assert lib.pm_beam_reorder(None, 0, None, 0, None, 2, 4, None) == L.PM_OK
    arr = (L.State * 1)(_state())
    assert lib.pm_beam_reorder(arr, 1, None, 0, None, 0, 4, None) == L.PM_OK


def test_beam_reorder_refuses_memory_that_overlaps():
    """Dense tensors that share a part of their memory; the parts of one
    buffer that lie between one another do not."""
    parents = torch.zeros(1, 3, dtype=torch.int32)
    buf = torch.zeros(40)
    a, shifted, behind = buf[:12].view(3, 4), buf[4:16].view(3, 4), buf[12:24].view(3, 4)
    with pytest.raises(ValueError, match="overlap"):
        pm.beam_reorder([a, shifted], parents)
    with pytest.raises(ValueError, match="overlap"):
        pm.beam_reorder([a], parents, out=[shifted])
    with pytest.raises(ValueError, match="overlap"):
        pm.beam_reorder([a, torch.zeros(3, 4)], parents, out=[behind, buf[20:32].view(3, 4)])
    pair = torch.zeros(3, 2, 4)
    for states in ([a, behind], [pair[:, 0], pair[:, 1]]):
        with pytest.raises(ValueError, match="CUDA"):  # all that is left to refuse
            pm.beam_reorder(states, parents)
    with pytest.raises(ValueError, match="CUDA"):  # states that are only read may share
        pm.beam_reorder([a, shifted], parents, out=[torch.zeros(3, 4), torch.zeros(3, 4)])


def test_beam_reorder_refuses_a_state_with_a_gradient():
    parents = torch.zeros(1, 3, dtype=torch.int32)
    leaf = torch.zeros(3, 4, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        pm.beam_reorder([leaf], parents)
    with pytest.raises(ValueError, match="gradient"):
        pm.beam_reorder([torch.zeros(3, 4)], parents, out=[leaf])
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        pm.beam_reorder([leaf], parents)


def test_c_checks_of_alignment():
    lib = L.load()
    for bad in (dict(logits=0x1002), dict(logits=0x1001, dtype=1), dict(mask=0x2002, mask_stride=32)):
        assert lib.pm_top_logprobs(C.byref(_top(**bad)), 0x3000, 0x4000, None, None) == L.PM_ERR_ARG
        assert lib.pm_beam_select_workspace_bytes(C.byref(_beam(**bad))) == 0
    o = L.BeamOut()
    o.scores, o.parents, o.tokens = 0x6000, 0x7000, 0x8000
    assert lib.pm_beam_select(C.byref(_beam()), C.byref(o), 0x9008, 1 << 30, None) == L.PM_ERR_ARG


def test_beam_reorder_refuses_to_write_what_it_reads():
    """lengths or parents among the states: other states' moves read them."""
    parents = torch.zeros(2, 3, dtype=torch.int32)
    lengths = torch.ones(6, dtype=torch.int32)
    cache = torch.zeros(6, 5, 4)
    with pytest.raises(ValueError, match="share"):
        pm.beam_reorder([cache, lengths], parents, lengths=lengths, seq_dim=[1, None])
    with pytest.raises(ValueError, match="share"):
        pm.beam_reorder([parents.view(6, 1)], parents)
    with pytest.raises(ValueError, match="share"):
        pm.beam_reorder([torch.zeros(6, dtype=torch.int32)], parents, out=[lengths], lengths=lengths)
    with pytest.raises(ValueError, match="CUDA"):  # all that is left to refuse
        pm.beam_reorder([cache, lengths], parents, out=[torch.zeros_like(cache), torch.zeros_like(lengths)],
                        lengths=lengths, seq_dim=[1, None])
