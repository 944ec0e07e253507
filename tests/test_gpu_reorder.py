"""beam_reorder against a plain row-by-row form: bytes have to be equal."""

import numpy as np
import pytest
import torch

import beam_plain as P
import paged_moe_b200 as pm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _maps(rng, B, W, kind):
    if kind == "any":
        return rng.integers(0, W, (B, W))
    if kind == "permutation":
        return np.stack([rng.permutation(W) for _ in range(B)])
    if kind == "one":
        return np.repeat(rng.integers(0, W, (B, 1)), W, 1)
    if kind == "same":
        return np.tile(np.arange(W), (B, 1))
    return rng.integers(-2, W + 2, (B, W))  # "outside": some rows keep their own


def _fill(rng, shape, dtype):
    x = torch.from_numpy(rng.integers(-100, 100, shape).astype(np.float64))
    return x.to(dtype).to(DEV)


def _check(states, parents, lengths=None, dims=None, double=False):
    """Small whole numbers in every type, so that float64 holds them all."""
    par = torch.from_numpy(parents.astype(np.int32)).to(DEV)
    ln = None if lengths is None else torch.from_numpy(lengths.astype(np.int32)).to(DEV)
    before = [s.to(torch.float64).cpu().numpy() for s in states]
    out = None
    if double:
        out = [torch.full_like(s, 7) for s in states]
    dims = dims if dims is not None else [None] * len(states)
    got = pm.beam_reorder(states, par, out=out, lengths=ln, seq_dim=dims)
    torch.cuda.synchronize()
    for s, b, d, g in zip(states, before, dims, got):
        into = np.full_like(b, 7) if double else None
        want = P.reorder(b, parents, into, lengths if d is not None else None, d)
        np.testing.assert_array_equal(g.to(torch.float64).cpu().numpy(), want)
        if double:
            np.testing.assert_array_equal(s.to(torch.float64).cpu().numpy(), b)  # the sources stay


@pytest.mark.parametrize("double", [False, True])
@pytest.mark.parametrize("kind", ["any", "permutation", "one", "same", "outside"])
@pytest.mark.parametrize("B,W", [(1, 1), (3, 2), (2, 5), (1, 64), (7, 8)])
def test_maps(B, W, kind, double):
    rng = np.random.default_rng(1)
    R = B * W
    states = [_fill(rng, (R, 3, 70, 16), torch.bfloat16), _fill(rng, (R, 257), torch.int32),
              _fill(rng, (R,), torch.float32), _fill(rng, (R, 5), torch.uint8)]
    _check(states, _maps(rng, B, W, kind), double=double)


@pytest.mark.parametrize("double", [False, True])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("inner", [1, 3, 8, 65])
@pytest.mark.parametrize("offset", [0, 1])
def test_sizes_and_alignment(dtype, inner, offset, double):
    """Widths and bases of every alignment, runs of one element to several segments."""
    rng = np.random.default_rng(2)
    B, W = 2, 6
    states = []
    for n in (1, 2, 17, 1000, 6007):
        flat = torch.zeros(B * W * n * inner + offset, dtype=dtype, device=DEV)
        v = flat[offset:].view(B * W, n, inner)
        v.copy_(_fill(rng, (B * W, n, inner), dtype))
        states.append(v)
    _check(states, _maps(rng, B, W, "any"), double=double)


@pytest.mark.parametrize("double", [False, True])
@pytest.mark.parametrize("seq_dim", [1, 2])
@pytest.mark.parametrize("D", [1, 8, 33, 128])
def test_lengths(seq_dim, D, double):
    rng = np.random.default_rng(3)
    B, W, S, H = 4, 5, 300, 3
    shape = (B * W, S, H, D) if seq_dim == 1 else (B * W, H, S, D)
    states = [_fill(rng, shape, torch.bfloat16), _fill(rng, shape, torch.float32), _fill(rng, (B * W, 9), torch.int64)]
    lengths = rng.integers(0, S + 1, (B, W))
    lengths[0] = [0, 1, S, S + 50, -3]  # nothing, one, all, past the end, below zero
    _check(states, _maps(rng, B, W, "any"), lengths, [seq_dim, seq_dim, None], double=double)


def test_strided_states():
    rng = np.random.default_rng(4)
    B, W = 2, 4
    R = B * W
    big = _fill(rng, (R, 2, 3, 50, 16), torch.bfloat16)  # keys and values of one tensor
    keep = big.clone()
    par = _maps(rng, B, W, "any")
    k, v = big[:, 0], big[:, 1]
    _check([k, v], par)
    want = P.reorder(keep.double().cpu().numpy(), par)
    np.testing.assert_array_equal(big.double().cpu().numpy(), want)
    wide = _fill(rng, (R, 3, 64, 20), torch.float32)[:, :, :41, :]  # a cache with room behind its positions
    _check([wide], par)
    _check([wide], par, rng.integers(0, 42, (B, W)), [2])
    # a dense source into a strided double buffer, and back
    dense = _fill(rng, (R, 3, 41, 20), torch.float32)
    room = torch.zeros((R, 3, 64, 20), device=DEV)[:, :, :41, :]
    p = torch.from_numpy(par.astype(np.int32)).to(DEV)
    pm.beam_reorder(dense, p, out=room)
    np.testing.assert_array_equal(room.double().cpu().numpy(), P.reorder(dense.double().cpu().numpy(), par))
    back = torch.zeros_like(dense)
    pm.beam_reorder(room, p, out=back)
    np.testing.assert_array_equal(back.double().cpu().numpy(), P.reorder(room.double().cpu().numpy(), par))


def test_many_states_and_single():
    rng = np.random.default_rng(5)
    B, W = 2, 3
    _check([_fill(rng, (B * W, 4 + i), torch.float32) for i in range(150)], _maps(rng, B, W, "any"))
    t = _fill(rng, (B * W, 7), torch.float32)
    par = torch.tensor([[1, 1, 0], [2, 0, 1]], dtype=torch.int32, device=DEV)
    want = P.reorder(t.double().cpu().numpy(), par.cpu().numpy())
    got = pm.beam_reorder(t, par)
    assert got is t
    np.testing.assert_array_equal(t.double().cpu().numpy(), want)
    # parents as a slice of more candidates
    more = torch.tensor([[1, 1, 0, 2, 2], [2, 0, 1, 0, 0]], dtype=torch.int32, device=DEV)[:, :3]
    want = P.reorder(t.double().cpu().numpy(), more.cpu().numpy())
    pm.beam_reorder(t, more)
    np.testing.assert_array_equal(t.double().cpu().numpy(), want)
    empty = torch.zeros((6, 0), device=DEV)
    assert pm.beam_reorder(empty, par) is empty
    assert pm.beam_reorder([], par) == []


def test_offsets_past_32_bits():
    """A state whose rows start beyond 2^32 bytes."""
    rng = np.random.default_rng(6)
    t = torch.zeros((2, 2300 << 20), dtype=torch.uint8, device=DEV)
    t[1, :100] = 5
    t[1, -100:] = 9
    par = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    pm.beam_reorder(t, par)
    assert int(t[0, :100].sum()) == 500 and int(t[0, -100:].sum()) == 900 and int(t[1].max()) == 0
    assert int(t[0, 100:-100].max()) == 0
    ln = torch.tensor([[2 ** 31 - 1, 0]], dtype=torch.int32, device=DEV)
    pm.beam_reorder(t, torch.tensor([[0, 0]], dtype=torch.int32, device=DEV), lengths=ln, seq_dim=1)
    assert int(t[1, :100].sum()) == 500 and int(t[1, 2 ** 31:].max()) == 0


def test_captured_and_other_stream():
    rng = np.random.default_rng(7)
    B, W = 3, 4
    t = _fill(rng, (B * W, 2, 64, 32), torch.bfloat16)
    out = torch.zeros_like(t)
    par = torch.from_numpy(_maps(rng, B, W, "any").astype(np.int32)).to(DEV)
    pm.beam_reorder(t, par, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pm.beam_reorder(t, par, out=out)
    par.copy_(torch.from_numpy(_maps(rng, B, W, "permutation").astype(np.int32)))
    g.replay()
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out.double().cpu().numpy(),
                                  P.reorder(t.double().cpu().numpy(), par.cpu().numpy()))
    side = torch.cuda.Stream()
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pm.beam_reorder(t, par, out=out)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(out.double().cpu().numpy(),
                                  P.reorder(t.double().cpu().numpy(), par.cpu().numpy()))


def test_a_write_counts_as_one_in_place():
    """A tensor saved for a backward pass and reordered after it is refused by
    that pass, as any other write in place is."""
    state = torch.randn(4, 8, device=DEV)
    leaf = torch.randn(4, 8, device=DEV, requires_grad=True)
    parents = torch.tensor([[1, 0, 3, 2]], dtype=torch.int32, device=DEV)
    y = (state * leaf).sum()
    pm.beam_reorder([state], parents)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        inside = torch.randn(4, 8, device=DEV)
    before = inside.clone()
    pm.beam_reorder([inside], parents)
    assert torch.equal(inside, before[[1, 0, 3, 2]])
