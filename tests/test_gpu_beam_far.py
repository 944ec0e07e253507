"""top_logprobs and beam_select where logits divided by the temperature pass
2^20 in units of log 2: below it a row's sum counts in whole exponents, above
it in multiples of its own terms, and one row may hold both.

Tolerances are those of a log-probability anywhere else: the error of a term
e^(-d) depends on its distance d from the row's largest, not on where the row
lies.  With few different values the mean of d is at most log V, as there.
"""

import numpy as np
import pytest
import torch

import beam_plain as P
import paged_moe_b200 as pm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
LSE_TOL = 7.7e-6
EDGE = 2.0 ** 20
STEPS = [-5000.0, -4097.0, -4095.0, -3000.0, -40.0, -1.0, 1.0, 40.0, 4095.0, 4097.0, 5000.0]


def _at(exponent, temp):
    """The logit whose e^(x / T) is 2^exponent."""
    return exponent * temp * np.log(2.0)


def _rows(V, dtype, temp, kinds):
    """One row for each distance from -2^20 and from 2^20.  "one": a single
    token there, the rest far below; "half": every second token a little or a
    lot lower; "wide": levels up to 12 temperatures below it, a tenth far below."""
    rng = np.random.default_rng(3)
    rows = []
    for kind in kinds:
        for edge in (-EDGE, EDGE):
            for step in STEPS:
                top = _at(edge + step, temp)
                x = np.full(V, top)
                if kind == "one":
                    x[:] = -1.0e9 * temp
                    x[V // 3] = top
                elif kind == "half":
                    x[::2] = top - temp * rng.choice([3.0, 2000.0, 9000.0])
                else:
                    x -= temp * rng.integers(0, 13, V)
                    x[rng.random(V) < 0.1] = -3.0e9 * temp
                    x[V - 1] = top
                rows.append(x)
    return torch.from_numpy(np.stack(rows)).to(dtype)


def _close(got, want):
    got = got.double().cpu().numpy()
    np.testing.assert_array_equal(np.isneginf(got), np.isneginf(want))
    fin = np.isfinite(want)
    off = np.abs(got[fin] - want[fin]) - LSE_TOL - np.abs(want[fin]) * 2.0 ** -24
    assert (off <= 0).all(), off.max()


def _check(x, k, temp, words=None, repeat=1):
    """Rows repeated until no row is split over CTAs, or once for those that are."""
    V = x.shape[1]
    allowed = None if words is None else P.allowed_bits(words, V)
    mask = None if words is None else torch.from_numpy(words.view(np.int32)).to(DEV).repeat(repeat, 1)
    got = pm.top_logprobs(x.to(DEV).repeat(repeat, 1), k, temp=temp, mask=mask, return_lse=True)
    ids, lp, lse = P.top_logprobs(x.double().numpy(), k, temp, allowed)
    n = x.shape[0]
    for first in {0, (repeat - 1) * n}:
        np.testing.assert_array_equal(got["ids"][first:first + n].cpu().numpy(), ids)
        _close(got["logprobs"][first:first + n], lp)
        _close(got["lse"][first:first + n], lse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temp", [1.0, 0.7, 0.001, 40.0])
@pytest.mark.parametrize("V,repeat", [(700, 1), (9001, 6), (40000, 1)])
def test_top_near_the_edge(V, repeat, temp, dtype):
    _check(_rows(V, dtype, temp, ["one", "half", "wide"]), 12, temp, repeat=repeat)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temp", [1.0, 0.7])
def test_top_near_the_edge_with_a_mask_and_as_keys(temp, dtype):
    """Tokens that are gathered, and rows whose every element becomes a key."""
    x = _rows(3000, dtype, temp, ["half", "wide"])
    keep = np.random.default_rng(5).random(x.shape) < 0.03
    keep[:, [0, 1, 1000, 2999]] = True
    _check(x, 9, temp, words=P.pack_bits(keep))
    _check(x, 200, temp)


@pytest.mark.parametrize("temp", [1.0, 0.7, 0.001])
@pytest.mark.parametrize("repeat", [1, 30])
def test_top_parts_on_both_sides(repeat, temp):
    """Rows of nine tiles, some of whose parts lie above the edge and some
    below it, close enough together for all to count."""
    V, tile = 70001, 8192
    rng = np.random.default_rng(6)
    rows = []
    for edge in (-EDGE, EDGE):
        for step in (-30.0, -2.0, 0.0, 2.0, 30.0, 4096.0):
            for lead in range(0, 9, 4):  # the part that holds the largest
                x = _at(edge + step, temp) - temp * rng.integers(0, 9, V).astype(np.float64)
                x[lead * tile + 5] += 4 * temp
                x[(lead + 3) % 9 * tile + 9:][:3000] = -2.0e9 * temp
                rows.append(x)
    _check(torch.from_numpy(np.stack(rows)).float(), 20, temp, repeat=repeat)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["one", "wide"])
def test_select_near_the_edge(kind, dtype):
    """Beams on either side of the edge are ranked by what is left of them."""
    V, W = 5000, 4
    x = _rows(V, dtype, 1.0, [kind])[:20].view(-1, W, V)
    scores = -np.random.default_rng(7).random(x.shape[:2]).astype(np.float32)
    got = pm.beam_select(x.to(DEV), torch.from_numpy(scores).to(DEV), n=W)
    want = P.beam_select(x.double().numpy(), scores, W)
    _close(got["scores"], want[0])
    np.testing.assert_array_equal(got["parents"].cpu().numpy(), want[1])
    np.testing.assert_array_equal(got["tokens"].cpu().numpy(), want[2])
