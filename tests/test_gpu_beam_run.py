"""The operators together, as they are used: beams decoded step by step with
their states moved, and a draft head's gradient from the teacher's targets
along the decoded tokens.

The teacher is a small recurrent model whose fp32 logits feed both the package
and a 64-bit beam search in numpy, so that only the operators differ.  A step's
scores are off by at most the tolerance of one log-probability (7.7e-6 and half
a step of fp32); they add up over the steps.
"""

import numpy as np
import pytest
import torch

import beam_plain as P
import distill_plain as D
import paged_moe_b200 as pm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
STEP_TOL = 7.7e-6


class Teacher:
    """h' = tanh(h R + E[token]); logits = h' O."""

    def __init__(self, V, H, seed):
        g = torch.Generator().manual_seed(seed)
        self.E = torch.randn((V, H), generator=g).to(DEV)
        self.R = (torch.randn((H, H), generator=g) / H ** 0.5).to(DEV)
        self.O = (torch.randn((H, V), generator=g) * 0.7).to(DEV)

    def step(self, h, tokens):
        h = torch.tanh(h @ self.R + self.E[tokens.long()])
        return h, h @ self.O


@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("alpha", [0.0, 0.7])
def test_beam_decode(slots, alpha):
    B, W, V, H, steps, eos = 3, 4, 2003, 32, 9, 11
    m = Teacher(V, H, 1)
    rng = np.random.default_rng(2)
    h = torch.from_numpy(rng.standard_normal((B * W, H))).float().to(DEV)
    cache = torch.zeros((B * W, 2, steps, 8), dtype=torch.bfloat16, device=DEV)  # what each beam wrote at each step
    hist = torch.full((B * W, steps), -1, dtype=torch.int32, device=DEV)
    tokens = torch.from_numpy(rng.integers(0, V, B * W).astype(np.int32)).to(DEV)
    scores = torch.full((B, W), float("-inf"), device=DEV)
    scores[:, 0] = 0.0
    done = torch.zeros((B, W), dtype=torch.bool, device=DEV)
    lengths = torch.zeros((B, W), dtype=torch.int32, device=DEV)
    ref = dict(s=scores.double().cpu().numpy(), d=done.cpu().numpy(), n=lengths.cpu().numpy(), h=hist.cpu().numpy(),
               c=cache.double().cpu().numpy())
    for t in range(steps):
        h, x = m.step(h, tokens.clamp(min=0))
        x[:, eos] += 4.0 if t > 2 else 0.0  # some beams end
        cache[:, :, t, :] = tokens.view(-1, 1, 1).to(torch.bfloat16) % 64
        ref["c"][:, :, t, :] = cache[:, :, t, :].double().cpu().numpy()
        out = pm.beam_select(x.view(B, W, V), scores, n=W, done=done, eos=eos, lengths=lengths, length_penalty=alpha,
                             keep_slots=slots)
        so_far = torch.full((B * W,), t + 1, dtype=torch.int32, device=DEV)
        pm.beam_reorder([h, hist, cache], out["parents"], lengths=so_far, seq_dim=[None, None, 2])
        scores, tokens, done, lengths = out["scores"], out["tokens"].reshape(-1), out["done"], out["lengths"]
        hist[:, t] = tokens
        # the same step in 64 bits on the same logits
        S, Pa, T, Ln, Dn = P.beam_select(x.double().cpu().numpy().reshape(B, W, V), ref["s"], W, done=ref["d"], eos=eos,
                                         lengths=ref["n"], alpha=alpha, keep_slots=slots)
        np.testing.assert_array_equal(out["parents"].cpu().numpy(), Pa)
        np.testing.assert_array_equal(out["tokens"].cpu().numpy(), T)
        np.testing.assert_array_equal(out["done"].cpu().numpy(), Dn)
        np.testing.assert_array_equal(out["lengths"].cpu().numpy(), Ln)
        fin = np.isfinite(S)
        assert (np.abs(out["scores"].double().cpu().numpy()[fin] - S[fin])
                <= (t + 1) * (STEP_TOL + np.abs(S[fin]) * 2.0 ** -24)).all()
        ref["h"] = P.reorder(ref["h"], Pa)
        ref["c"] = P.reorder(ref["c"], Pa, lengths=np.full((B, W), t + 1), seq_dim=2)
        ref["h"][:, t] = T.reshape(-1)
        ref.update(s=S, d=Dn, n=Ln)
        np.testing.assert_array_equal(hist.cpu().numpy(), ref["h"])
        np.testing.assert_array_equal(cache.double().cpu().numpy(), ref["c"])
    assert ref["d"].any() and not ref["d"].all()


def test_teacher_targets_train_a_draft_head():
    """top_logprobs of the teacher's rows are distill_loss's targets; the
    gradient of a linear draft head against the formula's."""
    N, V, H, K, temp = 24, 5003, 48, 32, 1.5
    rng = np.random.default_rng(3)
    teacher = torch.from_numpy(rng.standard_normal((N, V)) * 3).to(torch.bfloat16).to(DEV)
    top = pm.top_logprobs(teacher, K, temp=temp)
    hid = torch.from_numpy(rng.standard_normal((N, H))).float().to(DEV)
    head = torch.from_numpy(rng.standard_normal((H, V)) * 0.2).float().to(DEV).requires_grad_()
    weights = torch.from_numpy(rng.random(N) < 0.8).float().to(DEV)
    for tail in ("drop", "bucket"):
        x = (hid.double() @ head.double()).float()
        loss = pm.distill_loss(x, top["ids"], top["logprobs"], temp=temp, tail=tail, weights=weights)
        (g,) = torch.autograd.grad(loss, head)
        xs = x.detach().double().cpu().numpy()
        want, gx, sizes = D.loss(xs, top["ids"].cpu().numpy(), top["logprobs"].cpu().numpy(), temp, tail,
                                 weights.cpu().numpy())
        assert abs(float(loss.detach()) - want) <= 2 * 1.1e-5 + abs(want) * 2.0 ** -24
        a = hid.double().cpu().numpy()
        gw = a.T @ gx
        # the loss's tolerance of each gradient element, through the head's product in 64 bits, and its rounding
        tol = np.abs(a).T @ (2.5 * 1.1e-5 * sizes + np.abs(gx) * 2.0 ** -23) + np.abs(gw) * 2.0 ** -23
        assert (np.abs(g.double().cpu().numpy() - gw) <= tol).all()
    # the targets are the teacher's own distribution: a student with its logits has no loss but the dropped mass
    ids, lp, _ = P.top_logprobs(teacher.double().cpu().numpy(), K, temp)
    np.testing.assert_array_equal(top["ids"].cpu().numpy(), ids)
    own = pm.distill_loss(teacher, top["ids"], top["logprobs"], temp=temp, tail="bucket", reduction="none")
    # each log q is off by at most the tolerance of a log-probability, on either side of the difference
    assert (own.abs() <= 4 * 1.1e-5 + 2.0 ** -20).all()
