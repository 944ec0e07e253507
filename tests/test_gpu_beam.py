"""top_logprobs and beam_select against plain 64-bit forms.

Tolerance of a log-probability x / T - lse.  lse = M / T + log S with S a sum
of terms e^(-d), d = (M - x) / T >= 0.  Each term is off by the rounding of
x - M, of the constant log2(e) / T and of their product (2.5 half steps of
2^-24 of d) and by the hardware exponential (2^-20 at most, the budget the
library's self-check holds it to); the mean of d under the softmax is at most
log V <= 12.5, so these move log S by at most 12.5 * 2.5 * 2^-24 + 2^-20
< 2.9e-6.  A thread adds 16 terms of a tile and then at most 64 tiles, each
sum off by half a step: 80 * 2^-24 < 4.8e-6; the joins after it are in 64
bits.  Together 7.7e-6, and half a step of the result: LSE_TOL + 2^-24 |lp|.
Ids and tokens have to be equal.
"""

import numpy as np
import pytest
import torch

import beam_plain as P
import paged_moe_b200 as pm
from paged_moe_b200 import workloads as W

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
LSE_TOL = 7.7e-6


def _close(got, want):
    got = got.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.isneginf(got), np.isneginf(want))
    fin = np.isfinite(want)
    assert (np.abs(got[fin] - want[fin]) <= LSE_TOL + np.abs(want[fin]) * 2.0 ** -24).all(), \
        np.abs(got[fin] - want[fin]).max()


def _logits(seed, rows, V, dtype, sigma=2.5, pad=0, offset=0):
    """[rows, V] on the device: peaked rows, `pad` elements between them,
    starting `offset` elements into the allocation."""
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(W.peaked_logits(rng, rows, V, sigma, 9.0, min(16, V))).to(dtype)
    store = torch.zeros(rows * (V + pad) + offset, dtype=dtype, device=DEV)
    view = store[offset:].view(rows, V + pad)[:, :V]
    view.copy_(x)
    return view


def _mask(seed, rows, V, share):
    return P.pack_bits(np.random.default_rng(seed).random((rows, V)) < share)


def _check_top(x, k, temp=1.0, words=None, per_row=True):
    mask = None
    allowed = None
    if words is not None:
        mask = torch.from_numpy(words.view(np.int32)).to(DEV)
        allowed = P.allowed_bits(np.broadcast_to(np.atleast_2d(words), (x.shape[0], np.atleast_2d(words).shape[1])),
                                 x.shape[1])
    got = pm.top_logprobs(x, k, temp=temp, mask=mask, return_lse=True)
    torch.cuda.synchronize()
    ids, lp, lse = P.top_logprobs(x.double().cpu().numpy(), k, temp, allowed)
    np.testing.assert_array_equal(got["ids"].cpu().numpy(), ids)
    _close(got["logprobs"], lp)
    # what fp32 cannot hold is infinite: from half a step behind its largest on
    _close(got["lse"], np.where(np.abs(lse) >= 2.0 ** 128 * (1 - 2.0 ** -25), np.sign(lse) * np.inf, lse))
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (1, 1, 5), (3, 7, 7), (2, 31, 40), (4, 1000, 1), (3, 4096, 256),
                                      (2, 4097, 17), (5, 32768, 50), (1, 262144, 256), (9, 151937, 20)])
def test_top_sizes(dtype, rows, V, k):
    _check_top(_logits(1, rows, V, dtype), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (8, 0), (0, 5), (8, 8), (13, 2)])
def test_top_strides_and_alignment(dtype, pad, offset):
    _check_top(_logits(2, 4, 9001, dtype, pad=pad, offset=offset), 30)


@pytest.mark.parametrize("temp", [0.25, 0.8, 1.7, 30.0])
def test_top_temperature(temp):
    _check_top(_logits(3, 3, 20000, torch.float32), 12, temp=temp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("share", [0.001, 0.02, 0.5, 1.0])
def test_top_mask(dtype, share):
    rows, V = 6, 30011
    words = _mask(4, rows, V, share)
    words[2] = 0  # nothing allowed
    words[3] = 0
    words[3, 900] = 1 << 7  # one token
    x = _logits(5, rows, V, dtype)
    x[1, ::2] = float("nan")  # NaN where the mask forbids it
    words[1] &= np.uint32(0xAAAAAAAA)
    _check_top(x, 33, words=words)


def test_top_one_mask_for_all_rows():
    _check_top(_logits(6, 5, 5000, torch.float32), 9, words=_mask(7, 1, 5000, 0.3)[0])


def test_top_ties_and_signed_zeros():
    x = torch.zeros((4, 9000), device=DEV)
    x[1] = -0.0
    x[1, 5000:] = 0.0
    x[2] = torch.arange(9000, device=DEV) % 7  # ties everywhere
    x[3, 4096:] = 3.0
    got = _check_top(x, 100)
    assert got["ids"][0].tolist() == list(range(100)) == got["ids"][1].tolist()


def test_top_infinities_and_nan():
    x = _logits(8, 7, 6000, torch.float32)
    x[0, 100:] = float("-inf")
    x[1] = float("-inf")
    x[2, 5999] = float("nan")
    x[3, 3] = float("inf")
    x[4, :] = torch.finfo(torch.float32).min
    x[5, 1:] = torch.finfo(torch.float32).min
    x[6, 0], x[6, 1] = torch.finfo(torch.float32).max, torch.finfo(torch.float32).min
    _check_top(x, 150)
    _check_top(x.to(torch.bfloat16), 150)


@pytest.mark.parametrize("kind", ["ascending", "descending", "one_block"])
def test_top_orders(kind):
    """Orders that meet the key buffer at its worst: every tile above the last."""
    V = 50000
    x = torch.linspace(-20, 20, V, device=DEV)[None].repeat(2, 1)
    if kind == "descending":
        x = x.flip(1).contiguous()
    if kind == "one_block":
        x = torch.full((2, V), -30.0, device=DEV)
        x[:, 20000:24096] = torch.linspace(0, 9, 4096, device=DEV)
    _check_top(x, 256)
    _check_top(x.contiguous(), 1)


def test_top_transposed_and_empty():
    x = _logits(9, 300, 40, torch.float32)
    _check_top(x.t(), 8)  # a stride of 1 along the rows: copied
    out = pm.top_logprobs(torch.empty((0, 50), device=DEV), 4, return_lse=True)
    assert out["ids"].shape == (0, 4) and out["lse"].shape == (0,)


def test_equal_rows_get_equal_bits():
    """The same row at every alignment and place: the same bits."""
    base = _logits(10, 1, 50021, torch.bfloat16)
    x = torch.zeros((9, 50022), dtype=torch.bfloat16, device=DEV)[:, :50021]
    x.copy_(base.expand(9, -1))
    got = pm.top_logprobs(x, 40, return_lse=True)
    one = pm.top_logprobs(base, 40, return_lse=True)
    for r in range(9):
        assert torch.equal(got["logprobs"][r], one["logprobs"][0]) and torch.equal(got["lse"][r], one["lse"][0])


def test_limits_raise():
    x = torch.zeros((2, 300), device=DEV)
    with pytest.raises(RuntimeError):
        pm.top_logprobs(x, 257)
    with pytest.raises(RuntimeError):
        pm.top_logprobs(torch.zeros((1, 262145), device=DEV), 2)
    with pytest.raises(RuntimeError):
        pm.beam_select(x, torch.zeros((1, 2), device=DEV), n=257)
    with pytest.raises(RuntimeError):
        pm.beam_select(torch.zeros((1, 65, 10), device=DEV), torch.zeros((1, 65), device=DEV), n=2)
    with pytest.raises(ValueError):
        pm.beam_select(x, torch.zeros((1, 2)), n=2)  # scores on the host


# ---------------------------------------------------------------------------
# beam_select
# ---------------------------------------------------------------------------
def _check_select(x, scores, n, words=None, done=None, eos=None, lengths=None, alpha=0.0, slots=False):
    B, Wb = scores.shape
    dev = lambda a, t: None if a is None else torch.from_numpy(a).to(t).to(DEV)  # noqa: E731
    got = pm.beam_select(x, dev(scores, torch.float32), n=n, eos=eos, done=dev(done, torch.bool),
                         mask=None if words is None else torch.from_numpy(words.view(np.int32)).to(DEV),
                         lengths=dev(lengths, torch.int32), length_penalty=alpha, keep_slots=slots)
    torch.cuda.synchronize()
    V = x.shape[-1]
    allowed = None if words is None else P.allowed_bits(words, V)
    want = P.beam_select(x.double().cpu().numpy().reshape(B, Wb, V), scores.astype(np.float32), n, allowed, done,
                         -1 if eos is None else eos, lengths, alpha, slots)
    np.testing.assert_array_equal(got["parents"].cpu().numpy(), want[1])
    np.testing.assert_array_equal(got["tokens"].cpu().numpy(), want[2])
    _close(got["scores"], want[0])
    if lengths is not None:
        np.testing.assert_array_equal(got["lengths"].cpu().numpy(), want[3])
    else:
        assert "lengths" not in got
    if eos is not None:
        np.testing.assert_array_equal(got["done"].cpu().numpy(), want[4])
    return got


def _scores(seed, B, Wb):
    return (-np.random.default_rng(seed).random((B, Wb)) * 6).astype(np.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,Wb,V,n", [(1, 1, 1, 1), (1, 1, 2, 5), (2, 3, 50, 6), (1, 4, 32768, 8), (3, 5, 20011, 10),
                                      (2, 33, 5000, 40), (1, 64, 1000, 64), (1, 2, 262144, 256), (1, 64, 300, 256),
                                      (40, 2, 700, 3)])
def test_select_sizes(dtype, B, Wb, V, n):
    x = _logits(20, B * Wb, V, dtype).view(B, Wb, V)
    _check_select(x, _scores(21, B, Wb), n)


def test_select_first_step_has_one_beam():
    B, Wb, V = 3, 4, 9000
    s = np.full((B, Wb), -np.inf, dtype=np.float32)
    s[:, 0] = 0.0
    s[2] = -np.inf  # an item without any
    x = _logits(22, B * Wb, V, torch.float32)
    got = _check_select(x, s, 8)
    assert (got["parents"][:2] == 0).all() and (got["parents"][2] == -1).all()


@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("alpha", [0.0, 0.6, 1.0, -0.5])
def test_select_finished_beams(alpha, slots):
    B, Wb, V = 6, 5, 12001
    rng = np.random.default_rng(23)
    x = _logits(24, B * Wb, V, torch.bfloat16).view(B, Wb, V)
    done = rng.random((B, Wb)) < 0.4
    done[1] = True
    done[2] = False
    x[0][torch.from_numpy(done[0]).to(DEV)] = float("nan")  # their logits are not read
    lengths = rng.integers(0, 50, (B, Wb)).astype(np.int32)
    _check_select(x, _scores(25, B, Wb), Wb, done=done, eos=17, lengths=lengths, alpha=alpha, slots=slots)
    _check_select(x, _scores(26, B, Wb), Wb, done=done, eos=17, lengths=lengths, alpha=alpha, slots=slots)


def test_select_token_that_ends():
    x = torch.zeros((1, 2, 100), device=DEV)
    x[0, 0, 7] = 20.0
    x[0, 1, 8] = 20.0
    got = _check_select(x, np.zeros((1, 2), np.float32), 4, eos=7)
    assert got["done"].tolist()[0][:2] == [True, False]


@pytest.mark.parametrize("slots", [False, True])
def test_select_masks_and_bad_rows(slots):
    B, Wb, V = 4, 6, 8003
    x = _logits(27, B * Wb, V, torch.float32).view(B, Wb, V)
    words = _mask(28, B * Wb, V, 0.05)
    words[0:Wb] = 0  # item 0: nothing allowed anywhere
    words[Wb] = 0  # item 1: one beam without a token
    words[Wb + 1] = 0
    words[Wb + 1, 3] = 1 << 4  # and one with a single token
    x[2, 0, :] = float("nan")
    x[2, 1, :] = float("-inf")
    x[2, 2, :] = float("inf")
    x[3, 0, :] = torch.finfo(torch.float32).min
    _check_select(x, _scores(29, B, Wb), Wb, words=words, slots=slots)


def test_select_ties_go_to_the_lower_beam_and_token():
    x = torch.zeros((2, 3, 5000), device=DEV)
    x[1, :, 4999] = 1.0
    got = _check_select(x, np.zeros((2, 3), np.float32), 6)
    assert got["parents"][0].tolist() == [0] * 6 and got["tokens"][0].tolist() == list(range(6))
    assert got["parents"][1].tolist() == [0, 1, 2, 0, 0, 0]


def test_select_strides():
    for dtype, pad, offset in ((torch.bfloat16, 1, 3), (torch.float32, 2, 1)):
        x = _logits(30, 12, 7001, dtype, pad=pad, offset=offset)
        _check_select(x, _scores(31, 3, 4), 8)
    x = _logits(32, 12, 640, torch.float32).view(3, 4, 640).transpose(0, 1)  # [4, 3, V], beams not adjacent
    _check_select(x, _scores(33, 4, 3), 6)


def test_select_on_another_stream_and_captured():
    B, Wb, V = 4, 4, 30000
    x = _logits(34, B * Wb, V, torch.float32)
    s = torch.from_numpy(_scores(35, B, Wb)).to(DEV)
    want = pm.beam_select(x, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = pm.beam_select(x, s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same call, replayed at the same time
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pm.beam_select(x, s))
        graphs.append(g)
    for _ in range(5):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for got in (other, *outs):
        for k in want:
            assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k", [(2, 3000, 256), (3, 4096, 200), (64, 151936, 256), (5, 8192, 256), (1, 9000, 130),
                                      (7, 20000, 256)])
def test_top_large_k_of_short_parts(rows, V, k, dtype):
    """Few maxima for many candidates: rows, or parts of split rows, of one or two tiles."""
    _check_top(_logits(40, rows, V, dtype), k)


def test_top_short_parts_with_ties():
    x = torch.zeros((3, 6000), device=DEV)
    x[1, ::3] = 1.0
    x[2, 5000:] = 2.0
    _check_top(x, 256)
    _check_top(x.to(torch.bfloat16), 200)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k,allowed", [
    (3, 151937, 64, 3000), (2, 8192, 256, 682), (2, 8192, 256, 683), (2, 8192, 256, 684), (700, 40001, 130, 800),
    (400, 163840, 20, 3605), (400, 163840, 20, 3606), (3, 70001, 5, 0), (3, 70001, 5, 3)])
def test_top_few_allowed(dtype, rows, V, k, allowed):
    """Masks of an exact number of tokens, on both sides of where a part's
    tokens are gathered, the last token and the first among them; bits behind
    the vocabulary are set."""
    rng = np.random.default_rng(rows + V + allowed)
    keep = np.zeros((8, V), dtype=bool)
    for r in range(8):
        at = [0, V - 1][:allowed]
        keep[r, np.concatenate([at, rng.permutation(np.arange(1, V - 1))[:max(allowed - 2, 0)]]).astype(np.int64)] = True
    words = P.pack_bits(np.pad(keep, ((0, 0), (0, -V % 32)), constant_values=True))
    base = _logits(7, 8, V, dtype)
    x = base.repeat((rows + 7) // 8, 1)[:rows].contiguous()
    mask = torch.from_numpy(words.view(np.int32)).to(DEV).repeat((rows + 7) // 8, 1)[:rows].contiguous()
    got = pm.top_logprobs(x, k, mask=mask, return_lse=True)
    n = min(8, rows)
    ids, lp, lse = P.top_logprobs(base[:n].double().cpu().numpy(), k, 1.0, keep[:n])
    for first in (0, (rows - n) // 8 * 8):
        np.testing.assert_array_equal(got["ids"][first:first + n].cpu().numpy(), ids)
        _close(got["logprobs"][first:first + n], lp)
        _close(got["lse"][first:first + n], lse)


@pytest.mark.parametrize("B,Wb,n,slots", [(2, 21, 21, True), (2, 21, 30, False), (3, 64, 64, True), (1, 5, 256, False)])
@pytest.mark.parametrize("alpha", [0.0, 0.8])
def test_select_more_than_256_candidates(B, Wb, n, slots, alpha):
    """Lists merged in pairs: beams with the same logits and scores, ended and
    missing beams, rows with fewer allowed tokens than candidates."""
    rng = np.random.default_rng(60)
    V = 700
    x = _logits(61, B * Wb, V, torch.float32).view(B, Wb, V)
    x[:, 2] = x[:, 1]
    x[0, Wb - 1] = x[0, 0]
    x[B - 1, 3] = float("-inf")
    x[B - 1, 3, 9] = 1.0
    s = _scores(62, B, Wb)
    s[:, 2] = s[:, 1]
    s[0, Wb - 1] = s[0, 0]
    s[B - 1, 4] = -np.inf
    done = rng.random((B, Wb)) < 0.2
    done[:, :3] = False
    lengths = rng.integers(1, 40, (B, Wb)).astype(np.int32)
    lengths[:, 2] = lengths[:, 1]
    lengths[0, Wb - 1] = lengths[0, 0]
    _check_select(x, s, n, done=done, eos=5, lengths=lengths, alpha=alpha, slots=slots)
    _check_select(x, np.full_like(s, -np.inf), n, done=done, eos=5, lengths=lengths, alpha=alpha, slots=slots)
    words = _mask(63, B * Wb, V, 0.01)
    _check_select(x, s, n, words=words, lengths=lengths, alpha=alpha, slots=slots)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k,share", [
    (3, 1024, 32, None), (3, 1024, 33, None), (3, 1025, 64, None), (3, 1025, 65, None), (700, 4597, 161, None),
    (2, 7169, 256, None), (2, 7168, 225, None), (2, 7168, 224, 0.5), (2, 7168, 225, 0.5), (3, 1, 1, None), (5, 40, 256, 0.3)])
def test_top_more_wanted_than_threads_hold(dtype, rows, V, k, share):
    """Both sides of where every element of a short row becomes a key, with
    ties, infinities and offsets."""
    x = _logits(70, min(rows, 9), V, dtype, pad=3, offset=1)
    if V > 100:
        x[0, 10:90] = x[0, 5]
        x[1, ::2] = float("-inf")
        x[2 % x.shape[0], :] = torch.finfo(dtype).min
    if rows > x.shape[0]:
        big = torch.zeros(rows, V + 1, dtype=dtype, device=DEV)[:, :V]
        big.copy_(x.repeat((rows + 8) // 9, 1)[:rows])
        got = pm.top_logprobs(big, k)
        ids, lp, _ = P.top_logprobs(x.double().cpu().numpy(), k)
        for first in (0, (rows - 9) // 9 * 9):
            np.testing.assert_array_equal(got["ids"][first:first + 9].cpu().numpy(), ids)
            _close(got["logprobs"][first:first + 9], lp)
        return
    _check_top(x, k, temp=0.9, words=None if share is None else _mask(71, x.shape[0], V, share))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [900, 30000])
def test_rows_at_the_lowest_value_are_uniform(dtype, V):
    """All tokens at the type's lowest value, or far from zero: log V is not
    lost next to the logits."""
    x = torch.full((3, V), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    x[1] = 2.0 ** 60
    x[2] = -70000.0
    for temp in (1.0, 0.7):
        lp = pm.top_logprobs(x, 4, temp=temp)["logprobs"].double().cpu().numpy()
        assert (np.abs(lp + np.log(V)) <= LSE_TOL + np.log(V) * 2.0 ** -24).all(), lp
    got = pm.beam_select(x.view(1, 3, V), torch.tensor([[-1.0, -2.0, -3.0]], device=DEV), n=4)
    assert got["parents"].tolist() == [[0, 0, 0, 0]] and got["tokens"].tolist() == [[0, 1, 2, 3]]
    assert (np.abs(got["scores"].double().cpu().numpy() + 1 + np.log(V)) <= LSE_TOL + 12 * 2.0 ** -24).all()
