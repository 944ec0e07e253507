"""distill_loss and its gradient against a plain 64-bit form.

Tolerances.  With d = (M - x) / T >= 0, a term e^(-d) is off by 2.5 half
steps of 2^-24 of d (x - M, the constant log2(e) / T, their product) and by
the hardware exponential, 2^-20 at most.  Under the softmax the mean of d is
at most log V <= 12.5, which moves log S by 12.5 * 2.5 * 2^-24 + 2^-20 <
2.9e-6; fp32 sums of at most 132 terms in a row (8 of a vector, 124 to 128
vectors, then 64 bits) by 132 * 2^-24 < 7.9e-6.  So log S and log Q (the sum
outside the entries) are each off by less than REL = 1.1e-5, and a loss, in
which they enter with weights of at most 1 each, by 2 REL and half a step of
fp32.  A gradient's term q is off by REL, by its own e^(-d) (d <= 40 counts:
40 * 2.5 * 2^-24 + 2^-20 < 7e-6; smaller terms vanish) and three roundings;
q p_t / q_t by one more REL: 2.5 * REL of the terms' sizes together, and half
a step of the result's type (two where the loss's gradient is applied to the
rounded one).
"""

import numpy as np
import pytest
import torch

import distill_plain as P
import paged_moe_b200 as pm
from paged_moe_b200 import workloads as W

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
REL = 1.1e-5


def _case(seed, N, V, K, dtype=torch.float32, temp=1.0, pad=0, offset=0, ragged=False):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(W.peaked_logits(rng, N, V, 2.5, 9.0, min(16, V)))
    teacher = x + torch.from_numpy(rng.standard_normal((N, V)).astype(np.float32))
    lp = torch.log_softmax(teacher.double() / temp, 1)
    k = min(K, V)
    lps, ids = torch.topk(lp, k, dim=1)
    lps, ids = lps.float(), ids.to(torch.int32)
    if k < K:
        lps = torch.nn.functional.pad(lps, (0, K - k), value=0.0)
        ids = torch.nn.functional.pad(ids, (0, K - k), value=-1)
    if ragged:
        have = torch.from_numpy(rng.integers(0, K + 1, (N, 1)))
        ids = torch.where(torch.arange(K) < have, ids, -1)
    store = torch.zeros(N * (V + pad) + offset, dtype=dtype, device=DEV)
    view = store[offset:].view(N, V + pad)[:, :V]
    view.copy_(x.to(dtype))
    return view, ids.to(DEV), lps.to(DEV)


def _check_loss(got, want):
    got = got.detach().double().cpu().numpy()
    assert (np.abs(got - want) <= 2 * REL + np.abs(want) * 2.0 ** -24).all(), np.abs(got - want).max()


def _check_grad(got, want, sizes, roundings=1):
    eps = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu().numpy()
    tol = 2.5 * REL * sizes + np.abs(want) * (1.02 * roundings * eps) + 1e-37
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def _check(x, ids, lps, temp=1.0, tail="drop", weights=None, reduction="mean", up=None):
    w = None if weights is None else torch.from_numpy(weights.astype(np.float32)).to(DEV)
    wf = None if weights is None else weights.astype(np.float32)
    kw = dict(temp=temp, tail=tail, weights=w, reduction=reduction)
    want, grad, sizes = P.loss(x.double().cpu().numpy(), ids.cpu().numpy(), lps.float().cpu().numpy(), temp, tail, wf,
                               reduction, up)
    _check_loss(pm.distill_loss(x, ids, lps, **kw), want)
    leaf = x.detach().requires_grad_()
    loss = pm.distill_loss(leaf, ids, lps, **kw)
    _check_loss(loss, want)
    g = None
    if up is not None:
        g = torch.tensor(up, dtype=torch.float32, device=DEV)
    (got,) = torch.autograd.grad(loss, leaf, g)
    torch.cuda.synchronize()
    assert got.dtype == x.dtype and got.shape == x.shape
    _check_grad(got, grad, sizes, 2 if up is not None and reduction != "none" else 1)
    return got


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (1, 2, 1), (2, 5, 8), (3, 33, 33), (1, 4096, 256), (5, 8193, 20),
                                   (2, 32768, 64), (1, 262144, 256), (3, 151937, 50), (40, 700, 7)])
def test_sizes(N, V, K, dtype, tail):
    x, ids, lps = _case(1, N, V, K, dtype)
    _check(x, ids, lps, tail=tail)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reductions_weights_and_upstream(dtype, reduction, tail):
    rng = np.random.default_rng(2)
    x, ids, lps = _case(3, 9, 10007, 12, dtype, ragged=True)
    w = rng.random(9)
    w[[0, 4]] = 0.0
    w[5] = -0.5
    up = rng.standard_normal(9) if reduction == "none" else 0.37
    for weights in (None, w):
        for u in (None, up):
            if u is None and reduction == "none":
                u = np.ones(9)
            _check(x, ids, lps, tail=tail, weights=weights, reduction=reduction, up=u)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("temp", [0.5, 2.0, 7.0])
def test_temperature(temp, tail):
    x, ids, lps = _case(4, 3, 20000, 30, temp=temp)
    _check(x, ids, lps, temp=temp, tail=tail)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,offset", [(1, 0), (8, 0), (3, 1), (0, 5), (8, 8), (6, 2)])
def test_strides_and_alignment(dtype, pad, offset):
    x, ids, lps = _case(5, 4, 9001, 16, dtype, pad=pad, offset=offset)
    _check(x, ids, lps, tail="bucket")


def test_leading_dimensions_and_transposed():
    x, ids, lps = _case(6, 6, 500, 8)
    leaf = x.reshape(2, 3, 500).requires_grad_()
    loss = pm.distill_loss(leaf, ids.view(2, 3, 8), lps.view(2, 3, 8), reduction="none")
    assert loss.shape == (2, 3)
    (g,) = torch.autograd.grad(loss.sum(), leaf)
    want, grad, sizes = P.loss(x.double().cpu().numpy(), ids.cpu().numpy(), lps.cpu().numpy(), reduction="sum")
    _check_grad(g.reshape(6, 500), grad, sizes)
    leaf = x.t().contiguous().t().requires_grad_()
    (g,) = torch.autograd.grad(pm.distill_loss(leaf, ids.long(), lps, reduction="sum"), leaf)
    _check_grad(g, grad, sizes)


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_ids_twice_outside_and_none(tail):
    x, ids, lps = _case(7, 6, 3001, 10)
    lps = lps - 1.0
    ids[0, 3] = ids[0, 1]
    ids[0, 9] = ids[0, 1]
    ids[1, 2], ids[1, 3] = 3001, -7  # outside
    ids[2] = -1  # a row without entries
    lps[3, 4:] = float("-inf")  # entries without mass
    lps[4] = float("-inf")
    lps[0, 5] = lps[0, 6]
    _check(x, ids, lps, tail=tail)
    _check(x.to(torch.bfloat16), ids, lps, tail=tail)


def test_ids_past_32_bits_are_no_entries():
    x, ids, lps = _case(8, 2, 100, 4)
    far = ids.long()
    far[0, 1] = 2 ** 32 + 5
    ids[0, 1] = -1
    a = pm.distill_loss(x, far, lps, reduction="none")
    assert torch.equal(a, pm.distill_loss(x, ids, lps, reduction="none"))


def test_ignored_rows_are_not_read():
    x, ids, lps = _case(9, 5, 2000, 6)
    x[1] = float("nan")
    ids[1] = 2 ** 30
    lps[1] = float("nan")
    w = np.array([1.0, 0.0, 2.0, 1.0, 0.5])
    clean = x.clone()
    clean[1] = 0
    for reduction in ("mean", "sum"):
        leaf = x.detach().requires_grad_()
        wt = torch.from_numpy(w.astype(np.float32)).to(DEV)
        loss = pm.distill_loss(leaf, ids, lps, weights=wt, reduction=reduction)
        (g,) = torch.autograd.grad(loss, leaf)
        assert (g[1] == 0).all() and torch.isfinite(g).all()
        want, grad, sizes = P.loss(clean.double().cpu().numpy(), ids.cpu().numpy(), lps.cpu().numpy(), 1.0, "drop", w,
                                   reduction)
        _check_loss(loss, want)
        _check_grad(g, grad, sizes)
    zero = torch.zeros(5, device=DEV)
    leaf = x.detach().requires_grad_()
    loss = pm.distill_loss(leaf, ids, lps, weights=zero)
    assert float(loss.detach()) == 0.0
    assert (torch.autograd.grad(loss, leaf)[0] == 0).all()


@pytest.mark.parametrize("tail", ["drop", "bucket"])
def test_extreme_logits(tail):
    x, ids, lps = _case(10, 4, 4000, 5)
    ids = ids.clamp(max=3999)
    x[0, 2000:] = float("-inf")
    ids[0] = torch.arange(5, device=DEV)
    x[1] = torch.finfo(torch.float32).min  # all equal, at the type's lowest value
    x[2, 7] = 3.0e38
    ids[2] = torch.arange(5, 10, device=DEV)
    x[2, 5:10] = 3.0e38
    x[3] = -1.0e30
    x[3, 100:] = 5.0
    ids[3] = torch.arange(200, 205, device=DEV)
    _check(x, ids, lps, tail=tail)


def test_no_distribution_is_nan():
    x, ids, lps = _case(11, 4, 500, 5)
    x[0] = float("-inf")
    x[1, 3] = float("nan")
    x[2, 3] = float("inf")
    loss = pm.distill_loss(x, ids, lps, reduction="none")
    assert torch.isnan(loss[:3]).all() and torch.isfinite(loss[3])


def test_bucket_of_a_student_without_tail():
    """All of the student's mass on the entries: the tail counts as 2^-100."""
    x, ids, lps = _case(12, 2, 300, 3)
    x[:] = -2000.0
    x.scatter_(1, ids.long(), torch.tensor([[3.0, 2.0, 1.0]], device=DEV).expand(2, 3))
    lps = torch.log(torch.tensor([[0.5, 0.2, 0.1]], device=DEV)).expand(2, 3)
    _check(x, ids, lps, tail="bucket")


def test_backward_runs_once_and_no_grad():
    x, ids, lps = _case(13, 3, 100, 4)
    leaf = x.detach().requires_grad_()
    loss = pm.distill_loss(leaf, ids, lps)
    loss.backward(retain_graph=True)
    first = leaf.grad.clone()
    with pytest.raises(RuntimeError, match="one backward"):
        loss.backward()
    assert torch.equal(leaf.grad, first)
    with torch.no_grad():
        assert not pm.distill_loss(leaf, ids, lps).requires_grad
    per = pm.distill_loss(leaf, ids, lps, reduction="none")
    a = torch.autograd.grad(per.sum(), leaf, retain_graph=True)[0]
    b = torch.autograd.grad(per.sum(), leaf)[0]
    assert torch.equal(a, b)


def test_gradient_accumulates_through_a_head():
    """The loss behind an LM head, as a draft head trains: gradients of the
    head's weight against the formula's."""
    rng = np.random.default_rng(14)
    h = torch.from_numpy(rng.standard_normal((12, 64))).float().to(DEV)
    w = torch.from_numpy(rng.standard_normal((900, 64)) * 0.3).float().to(DEV).requires_grad_()
    ids = torch.from_numpy(rng.integers(0, 900, (12, 6))).to(torch.int32).to(DEV)
    lps = torch.log(torch.from_numpy(rng.dirichlet(np.ones(6), 12) * 0.9).float()).to(DEV)
    for _ in range(2):
        pm.distill_loss(h.double().matmul(w.double().t()).float(), ids, lps, tail="bucket").backward()
    x = h.double().cpu().numpy() @ w.detach().double().cpu().numpy().T
    _, g, sizes = P.loss(np.float64(np.float32(x)), ids.cpu().numpy(), lps.cpu().numpy(), tail="bucket")
    want = 2 * (g.T @ h.double().cpu().numpy())
    bound = 2 * ((2.5 * REL * sizes + np.abs(g) * 2.0 ** -23).T @ np.abs(h.double().cpu().numpy()))
    got = w.grad.double().cpu().numpy()
    assert (np.abs(got - want) <= bound + np.abs(want) * 2.0 ** -22).all()


def test_empty_batch():
    x = torch.empty((0, 50), device=DEV, requires_grad=True)
    ids, lps = torch.empty((0, 3), dtype=torch.int32, device=DEV), torch.empty((0, 3), device=DEV)
    loss = pm.distill_loss(x, ids, lps)
    assert float(loss.detach()) == 0.0
    assert torch.autograd.grad(loss, x)[0].shape == (0, 50)
    assert pm.distill_loss(x.detach(), ids, lps, reduction="none").shape == (0,)


def test_same_bits_every_time():
    x, ids, lps = _case(15, 7, 30011, 20, torch.bfloat16)
    w = torch.rand(7, device=DEV)
    runs = []
    for _ in range(3):
        leaf = x.detach().requires_grad_()
        loss = pm.distill_loss(leaf, ids, lps, weights=w, tail="bucket")
        runs.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
    for l, g in runs[1:]:
        assert torch.equal(l, runs[0][0]) and torch.equal(g, runs[0][1])


def test_another_stream_and_captured():
    x, ids, lps = _case(16, 6, 20000, 16, torch.bfloat16)
    leaf = x.detach().requires_grad_()
    loss = pm.distill_loss(leaf, ids, lps)
    (want,) = torch.autograd.grad(loss, leaf)
    want_loss = loss.detach().clone()
    del loss
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        l2 = pm.distill_loss(leaf, ids, lps)
        (g2,) = torch.autograd.grad(l2, leaf)
    torch.cuda.synchronize()
    assert torch.equal(g2, want) and torch.equal(l2.detach(), want_loss)
    del l2
    fresh = x.detach().clone().requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        l3 = pm.distill_loss(fresh, ids, lps)
        (g3,) = torch.autograd.grad(l3, fresh)
    with torch.no_grad():
        fresh.zero_()
        fresh.copy_(x)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(g3, want) and torch.equal(l3.detach(), want_loss)


def test_limits_raise():
    x = torch.zeros((2, 300), device=DEV)
    ids, lps = torch.zeros((2, 257), dtype=torch.int32, device=DEV), torch.zeros((2, 257), device=DEV)
    with pytest.raises(RuntimeError):
        pm.distill_loss(x, ids, lps)
    with pytest.raises(ValueError):
        pm.distill_loss(x, ids[:, :3].cpu(), lps[:, :3])


@pytest.mark.parametrize("dtype,N,V,pad,offset", [
    (torch.float32, 3, 16383, 1, 3), (torch.float32, 2, 16384, 0, 0), (torch.bfloat16, 2, 32767, 9, 7),
    (torch.bfloat16, 3, 100, 0, 1), (torch.float32, 1, 1, 0, 2), (torch.float32, 2, 40001, 2, 1)])
def test_a_loss_with_a_factor(dtype, N, V, pad, offset):
    """The factor multiplies the loss's gradient as it was stored, one
    rounding more; nothing beside the rows is written."""
    x, ids, lps = _case(40, N, V, 5, dtype, pad=pad, offset=offset)
    x.requires_grad_()
    plain = torch.autograd.grad(pm.distill_loss(x, ids, lps, reduction="sum"), x)[0]
    scaled = torch.autograd.grad(pm.distill_loss(x, ids, lps, reduction="sum") * 0.7, x)[0]
    # in fp32 here: a bf16 tensor times a tensor of no dimensions rounds 0.7 to bf16 first
    assert torch.equal(scaled, (plain.float() * np.float32(0.7).item()).to(dtype))
    grad = torch.full((N * (V + pad) + offset + 40,), 3.0, dtype=dtype, device=DEV)
    rows = grad[offset:offset + N * (V + pad)].view(N, V + pad)
    before = grad.clone()
    from paged_moe_b200 import _lib as L
    code = L.PM_DTYPE_F32 if dtype == torch.float32 else L.PM_DTYPE_BF16
    factor = torch.tensor([-0.5], device=DEV)
    L.check(L.load().pm_distill_scale(rows.data_ptr(), code, N, V, V + pad, factor.data_ptr(),
                                      torch.cuda.current_stream().cuda_stream), "pm_distill_scale")
    want = before.clone()
    want[offset:offset + N * (V + pad)].view(N, V + pad)[:, :V] *= -0.5
    assert torch.equal(grad, want)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_no_second_derivative(reduction):
    x, ids, lps = _case(41, 3, 100, 4)
    x.requires_grad_()
    up = torch.ones((), device=DEV, requires_grad=True)
    loss = (pm.distill_loss(x, ids, lps, reduction=reduction) * up).sum()
    grad = torch.autograd.grad(loss, x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second derivative"):
        grad.sum().backward()


@pytest.mark.parametrize("tail", ["drop", "bucket"])
@pytest.mark.parametrize("N,V,dtype", [(371, 60, torch.float32), (400, 8191, torch.bfloat16), (380, 4096, torch.float32),
                                       (2, 20011, torch.float32), (300, 5000, torch.bfloat16)])
def test_rows_that_need_care(N, V, dtype, tail):
    """Rows for a warp each and rows for CTAs and clusters: constant rows,
    rows far from zero, rows with few finite logits, ids twice, outside and
    none, weights of zero, one row on its own in the last CTA."""
    x, ids, lps = _case(50 + N, N, V, 7, dtype, pad=3, offset=1)
    x[0] = 2.0
    x[1] *= 1000.0
    if N > 2:
        x[2] = float("-inf")
        x[2, [0, V // 2, V - 1]] = torch.tensor([1.0, 2.0, 0.5], dtype=dtype, device=DEV)
        ids[2, :3] = torch.tensor([V - 1, 0, V // 2], dtype=torch.int32, device=DEV)  # an entry of no mass has an infinite loss
        ids[2, 3:] = -1
        x[3] -= 60000.0
        x[4] *= 3.0e6
        ids[5, 1] = ids[5, 0]
        ids[6] = -1
        ids[7, 2] = V
        ids[8, 3] = ids[8, 1] = ids[8, 0]
    lps = torch.log_softmax(lps, 1) - 0.1
    w = np.ones(N, dtype=np.float32)
    w[N // 2:N // 2 + 9] = 0.0
    w[N - 1] = 2.5
    _check(x, ids, lps, temp=1.3, tail=tail, weights=w, reduction="mean")
    _check(x, ids, lps, temp=1.3, tail=tail, weights=w, reduction="none", up=np.ones(N, dtype=np.float32))


def test_no_distribution_and_no_weight_on_both_sides():
    for N, V in ((400, 500), (3, 30011)):
        x, ids, lps = _case(60, N, V, 4)
        x[1] = float("-inf")
        x[2, 7] = float("nan")
        leaf = x.clone().requires_grad_()
        loss = pm.distill_loss(leaf, ids, lps, reduction="none")
        grad = torch.autograd.grad(loss.sum(), leaf)[0]
        assert torch.isnan(loss[1:3]).all() and torch.isnan(grad[1:3]).all()
        assert not torch.isnan(loss[0]) and not torch.isnan(grad[0]).any()
        zero = torch.zeros(N, device=DEV)
        for tail in ("drop", "bucket"):
            for reduction in ("mean", "sum"):
                loss = pm.distill_loss(leaf, ids, lps, weights=zero, tail=tail, reduction=reduction)
                assert float(loss.detach()) == 0.0
                assert not torch.autograd.grad(loss, leaf)[0].any()


def test_two_captured_graphs_of_many_short_rows_and_their_inputs_change():
    """Two graphs of the same leaf replayed in turn, with other logits each
    time: neither keeps anything of the other's or of its last run."""
    x, ids, lps = _case(70, 500, 900, 12)
    y = _case(71, 500, 900, 12)[0]
    w = torch.rand(500, device=DEV)
    w[::7] = 0.0
    leaf = x.detach().clone().requires_grad_()
    kinds = (dict(tail="bucket", weights=w), dict(tail="drop", reduction="sum", temp=0.5))
    graphs = []
    for kw in kinds:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss = pm.distill_loss(leaf, ids, lps, **kw)
            (grad,) = torch.autograd.grad(loss, leaf)
        graphs.append((g, loss, grad, kw))
    for source in (x, y, x):
        with torch.no_grad():
            leaf.copy_(source)
        for g, _, _, _ in graphs:
            g.replay()
        for _, loss, grad, kw in graphs:
            eager = source.detach().clone().requires_grad_()
            want = pm.distill_loss(eager, ids, lps, **kw)
            assert torch.equal(loss.detach(), want.detach())
            assert torch.equal(grad, torch.autograd.grad(want, eager)[0])


def test_same_bits_of_many_short_rows_and_on_two_streams_at_once():
    x, ids, lps = _case(72, 900, 3001, 20, torch.bfloat16)
    w = torch.rand(900, device=DEV)

    def run():
        leaf = x.detach().requires_grad_()
        loss = pm.distill_loss(leaf, ids, lps, weights=w, tail="bucket")
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for l, g in got:
        assert torch.equal(l, want[0]) and torch.equal(g, want[1])
