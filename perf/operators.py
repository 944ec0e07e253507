"""The operators around beam decoding and draft-model distillation: their
cases, inputs and plain forms.

Four operators, each a call of the package:

    top_logprobs   the k best tokens of every row with their log-probabilities
    beam_select    the n best continuations over beams and vocabulary
    beam_reorder   per-beam states moved to the beams that continue them
    distill_loss   KL loss from a teacher's top log-probabilities, and its gradient

With `own` false `run` computes them from elementary torch operations; with
`own` true it makes the calls a user's program makes.  `exact` states each
definition once more, row by row, in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
NEG = float("-inf")


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _top(name, rows, vocab, dtype, k, temp=1.0, mask=0.0, pad=0, lse=True):
    """mask: share of allowed tokens (0: no mask); pad: elements between rows."""
    return {"name": name, "op": "top", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "temp": temp,
            "mask": mask, "pad": pad, "lse": lse}


def _select(name, items, beams, vocab, dtype, n, mask=0.0, ended=0.0, penalty=0.0, slots=False, pad=0):
    """ended: share of finished beams; penalty: exponent of the length."""
    return {"name": name, "op": "select", "items": items, "beams": beams, "vocab": vocab, "dtype": dtype, "n": n,
            "mask": mask, "ended": ended, "penalty": penalty, "slots": slots, "pad": pad}


def _reorder(name, items, beams, states, heads, positions, width, dtype, seq_dim, in_place, ragged, history=0):
    """states: tensors [rows, heads, positions, width] (seq_dim 2) or [rows,
    positions, heads, width] (seq_dim 1); ragged: lengths from 1 to positions;
    history: width of one more int32 state, the token histories (0: none)."""
    return {"name": name, "op": "reorder", "items": items, "beams": beams, "states": states, "heads": heads,
            "positions": positions, "width": width, "dtype": dtype, "seq_dim": seq_dim, "in_place": in_place,
            "ragged": ragged, "history": history}


def _distill(name, rows, vocab, dtype, k, temp, tail, train, reduction="mean", weighted=False, ragged=False, pad=0):
    """train: the gradient too; weighted: row weights, some 0; ragged: rows
    with fewer than k teacher entries."""
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "temp": temp,
            "tail": tail, "train": train, "reduction": reduction, "weighted": weighted, "ragged": ragged, "pad": pad}


def listed():
    return [
        # the log-probabilities an API answers with, for the k + 1 rows of one verify pass
        _top("top_verify_rows", 5, 151552, "f32", 20),
        # constrained rows of a serving batch: an allowed-token mask, an odd vocabulary
        _top("top_masked_odd", 61, 151937, "bf16", 64, temp=0.8, mask=0.02),
        # a teacher's targets for 2,048 training positions
        _top("top_teacher", 2048, 163840, "bf16", 64),
        # one request decoding with 4 beams: latency counts
        _select("select_one", 1, 4, 32768, "f32", 8),
        # a batch with finished beams, length penalty and a mask, odd sizes, beams kept in their slots
        _select("select_ended_odd", 12, 5, 151937, "bf16", 5, mask=0.3, ended=0.3, penalty=0.6, slots=True),
        # a full batch of 8 beams, twice as many candidates as beams
        _select("select_batch", 64, 8, 163840, "f32", 16),
        # a small model's states after one short step: many launches if done one by one
        _reorder("reorder_small", 2, 4, 8, 4, 33, 64, "f32", 2, False, False, history=257),
        # odd widths and lengths, positions before heads, copied into the other half of a double buffer
        _reorder("reorder_odd", 16, 6, 6, 3, 1001, 65, "bf16", 1, False, True),
        # a long key-value cache in place, the beams that live on in their slots
        _reorder("reorder_cache", 4, 8, 8, 8, 2048, 128, "bf16", 2, True, True),
        # validation loss of a small vocabulary
        _distill("distill_eval", 16, 32768, "f32", 20, 1.0, "drop", False),
        # a training step on 2,048 positions, the teacher's remaining mass in one bucket
        _distill("distill_train", 2048, 163840, "bf16", 64, 1.0, "bucket", True),
        # a small step: fp32 logits, odd vocabulary, ignored rows, short teacher rows, temperature
        _distill("distill_train_odd", 257, 151937, "f32", 50, 2.0, "drop", True, weighted=True, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rows_vocab(rng, size, most_rows, most_bytes):
    vocab = _log_int(rng, 1000, 262144)
    rows = _log_int(rng, 1, max(1, min(most_rows, most_bytes // (vocab * size))))
    return rows, vocab


def draw(rng):
    op = rng.choice(["top", "select", "reorder", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    size = 4 if dtype == "f32" else 2
    pad = rng.choice([0, 0, 1, 8])
    if op == "top":
        rows, vocab = _rows_vocab(rng, size, 2048, 500 << 20)
        c = _top("", rows, vocab, dtype, _log_int(rng, 1, 256), temp=rng.choice([1.0, 0.7, 1.7]),
                 mask=rng.choice([0.0, 0.0, 0.02, 0.5]), pad=pad)
    elif op == "select":
        rows, vocab = _rows_vocab(rng, size, 512, 300 << 20)
        beams = min(rows, _log_int(rng, 1, 16))
        slots = rng.random() < 0.3
        n = beams if slots else _log_int(rng, 1, 4 * beams)
        c = _select("", max(1, rows // beams), beams, vocab, dtype, n, mask=rng.choice([0.0, 0.0, 0.1]),
                    ended=rng.choice([0.0, 0.25]), penalty=rng.choice([0.0, 0.0, 1.0]), slots=slots, pad=pad)
    elif op == "reorder":
        width = rng.choice([16, 64, 128, 65, 1])
        heads, positions = _log_int(rng, 1, 16), _log_int(rng, 1, 4096)
        one = heads * positions * width * size
        beams = _log_int(rng, 2, 16)
        items = _log_int(rng, 1, max(1, min(64, (60 << 20) // (one * beams))))
        states = _log_int(rng, 1, 16)
        c = _reorder("", items, beams, states, heads, positions, width, dtype, rng.choice([1, 2]),
                     rng.random() < 0.5, rng.random() < 0.6, history=rng.choice([0, 1, 300]))
    else:
        rows, vocab = _rows_vocab(rng, size, 2048, 300 << 20)
        c = _distill("", rows, vocab, dtype, _log_int(rng, 1, 256), rng.choice([1.0, 1.0, 2.0, 0.5]),
                     rng.choice(["drop", "bucket"]), rng.random() < 0.7, rng.choice(["mean", "sum", "none"]),
                     rng.random() < 0.4, rng.random() < 0.4, pad)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _peaked(g, rows, vocab, dtype, pad):
    """Logits as a language model's last step gives them: a broad bulk, 16
    ids per row well above it."""
    x = torch.randn((rows, vocab + pad), generator=g, device=DEV)
    x *= 2.5
    ids = torch.randint(0, vocab, (rows, 16), generator=g, device=DEV)
    x.scatter_add_(1, ids, 8.0 + 2.0 * torch.randn((rows, 16), generator=g, device=DEV))
    return x.to(_type(dtype))[:, :vocab]


def _mask(g, rows, vocab, share):
    """Packed allowed-token words [rows, ceil(vocab / 32)]."""
    words = (vocab + 31) // 32
    bits = (torch.rand((rows, words * 32), generator=g, device=DEV) < share).view(rows, words, 32)
    w = (bits.to(torch.int64) << torch.arange(32, device=DEV)).sum(-1)
    return (w - ((w >> 31) << 32)).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = {"case": case}
    op = case["op"]
    if op == "top":
        s["x"] = _peaked(g, case["rows"], case["vocab"], case["dtype"], case["pad"])
        s["mask"] = _mask(g, case["rows"], case["vocab"], case["mask"]) if case["mask"] else None
    elif op == "select":
        B, W, V = case["items"], case["beams"], case["vocab"]
        s["x"] = _peaked(g, B * W, V, case["dtype"], case["pad"])
        s["mask"] = _mask(g, B * W, V, case["mask"]) if case["mask"] else None
        s["eos"] = V - 1
        s["lengths"] = torch.randint(1, 200, (B, W), generator=g, device=DEV, dtype=torch.int32)
        s["scores"] = -0.5 * s["lengths"] - 2.0 * torch.rand((B, W), generator=g, device=DEV)
        s["done"] = (torch.rand((B, W), generator=g, device=DEV) < case["ended"]) if case["ended"] else None
    elif op == "reorder":
        B, W = case["items"], case["beams"]
        H, S, D = case["heads"], case["positions"], case["width"]
        shape = (B * W, H, S, D) if case["seq_dim"] == 2 else (B * W, S, H, D)
        # beams that live on keep their slots; the others take a living beam's state
        alive = torch.rand((B, W), generator=g, device=DEV) < 0.5
        alive.scatter_(1, torch.randint(0, W, (B, 1), generator=g, device=DEV), True)
        pick = torch.multinomial(alive.float(), W, replacement=True, generator=g)
        own_slot = torch.arange(W, device=DEV).expand(B, W)
        if not case["in_place"]:  # in rank order, as a selection gives them
            s["parents"] = torch.randint(0, W, (B, W), generator=g, device=DEV).to(torch.int32)
        else:
            s["parents"] = torch.where(alive, own_slot, pick).to(torch.int32)
        lengths = torch.randint(1, S + 1, (B, 1), generator=g, device=DEV, dtype=torch.int32).expand(B, W)
        s["lengths"] = lengths.contiguous() if case["ragged"] else None

        def states():
            t = [torch.randn(shape, generator=g, device=DEV).to(_type(case["dtype"])) for _ in range(case["states"])]
            if case["history"]:
                # the token histories, one column of ids per position of one head
                t.append(torch.randint(0, 32000, (B * W, case["history"]), generator=g, device=DEV, dtype=torch.int32))
            return t

        s["states"] = states()
        s["out"] = None if case["in_place"] else states()
    else:
        N, V, K = case["rows"], case["vocab"], case["k"]
        x = _peaked(g, N, V, case["dtype"], case["pad"])
        # the teacher: the student's logits in a sharper, shifted form
        t = torch.randn((N, V), generator=g, device=DEV)
        t += x
        t /= case["temp"]
        vals, ids = torch.topk(t, min(K, V), dim=1)
        s["lp"] = (vals - torch.logsumexp(t, dim=1, keepdim=True)).contiguous()
        del t
        s["ids"] = ids.to(torch.int32)
        if case["ragged"]:
            have = torch.randint(1, K + 1, (N, 1), generator=g, device=DEV)
            s["ids"] = torch.where(torch.arange(s["ids"].shape[1], device=DEV) < have, s["ids"], -1)
        s["weights"] = None
        if case["weighted"]:
            w = torch.rand((N,), generator=g, device=DEV)
            s["weights"] = torch.where(w < 0.25, torch.zeros_like(w), w)
        s["up"] = torch.randn((N,), generator=g, device=DEV)  # what flows back into a loss per row
        s["x"] = x.requires_grad_(True) if case["train"] else x
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _allowed(words, vocab):
    bits = (words[:, :, None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return bits.reshape(words.shape[0], -1)[:, :vocab].bool()


def _best(x, n):
    """The n largest values of each row and their ids, ties by the lowest id."""
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    key = (order << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
    ids = torch.topk(key, n, dim=1).indices
    return torch.gather(x, 1, ids), ids


def _row_lse(x, scale):
    """log of the sum of e^(x scale), the sum in 64 bits."""
    m = x.amax(1, keepdim=True)
    m = torch.where(m == NEG, torch.zeros_like(m), m)
    total = torch.exp((x - m) * scale).sum(1, dtype=torch.float64)
    return m.squeeze(1).double() * scale + torch.log(total)


def _plain_top(s):
    c = s["case"]
    x = s["x"].float()
    if s["mask"] is not None:
        x = x.masked_fill(~_allowed(s["mask"], c["vocab"]), NEG)
    lse = _row_lse(x, 1.0 / c["temp"])
    n = min(c["k"], c["vocab"])
    vals, ids = _best(x, n)
    gone = vals == NEG
    ids = ids.to(torch.int32).masked_fill(gone, -1)
    lp = (vals.double() / c["temp"] - torch.where(lse == NEG, torch.zeros_like(lse), lse)[:, None]).float()
    if n < c["k"]:
        ids = torch.nn.functional.pad(ids, (0, c["k"] - n), value=-1)
        lp = torch.nn.functional.pad(lp, (0, c["k"] - n), value=NEG)
    return {"ids": ids, "logprobs": lp, "lse": lse.float()}


def _plain_slots(parents):
    """Slot of each candidate of a ranked list: the parent's own for its best
    child, the free slots in ascending order for the rest."""
    B, n = parents.shape
    j = torch.arange(n, device=parents.device)
    earlier = j[None, :] < j[:, None]
    first = ~((parents[:, :, None] == parents[:, None, :]) & earlier).any(2) & (parents >= 0)
    taken = (first[:, None, :] & (parents[:, None, :] == j[None, :, None])).any(2)
    free = torch.argsort(taken.to(torch.int32), dim=1, stable=True)  # free slots first, ascending
    rest = torch.cumsum((~first).to(torch.int64), 1) - 1
    return torch.where(first, parents.to(torch.int64), torch.gather(free, 1, rest.clamp(min=0)))


def _plain_select(s):
    c = s["case"]
    B, W, V, n = c["items"], c["beams"], c["vocab"], c["n"]
    x = s["x"].float()
    if s["mask"] is not None:
        x = x.masked_fill(~_allowed(s["mask"], V), NEG)
    lse = _row_lse(x.double(), 1.0)  # 64 bits: totals of different beams may lie close together
    m = min(n, V)
    vals, ids = _best(x, m)
    score = s["scores"].reshape(-1).double()
    fit = (vals > NEG) & torch.isfinite(lse)[:, None] & (score > NEG)[:, None]
    total = torch.where(fit, score[:, None] + (vals.double() - torch.where(fit[:, :1], lse[:, None], 0.0)), NEG)
    length = s["lengths"].reshape(-1).to(torch.int64) + 1
    if s["done"] is not None:
        ended = s["done"].reshape(-1, 1)
        one = torch.where(torch.arange(m, device=x.device)[None, :] == 0, score[:, None], NEG)
        total = torch.where(ended, one, total)
        ids = torch.where(ended, s["eos"], ids)
        length = torch.where(ended[:, 0], length - 1, length)
    rank = total / length.clamp(min=1).double().pow(c["penalty"])[:, None]
    rank = rank.view(B, W * m)
    at = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :n]
    if at.shape[1] < n:  # fewer candidates than asked
        at = torch.nn.functional.pad(at, (0, n - at.shape[1]), value=-1)
    none = at < 0
    at = at.clamp(min=0)
    scores = torch.gather(total.view(B, -1), 1, at).masked_fill(none, NEG)
    none = none | (scores == NEG)
    parents = (at // m).masked_fill(none, -1)
    tokens = torch.gather(ids.reshape(B, -1), 1, at).masked_fill(none, -1)
    grown = torch.gather(length.view(B, W), 1, parents.clamp(min=0)).masked_fill(none, 0)
    done = tokens == s["eos"]
    if s["done"] is not None:
        done = done | (torch.gather(s["done"], 1, parents.clamp(min=0)) & ~none)
    out = {"scores": scores.float(), "parents": parents.to(torch.int32), "tokens": tokens.to(torch.int32),
           "lengths": grown.to(torch.int32), "done": done}
    if c["slots"]:
        slot = _plain_slots(out["parents"])
        out = {k: torch.empty_like(v).scatter_(1, slot, v) for k, v in out.items()}
    return out


def _plain_reorder(s):
    c = s["case"]
    B, W = c["items"], c["beams"]
    p = s["parents"].to(torch.int64)
    base = (torch.arange(B, device=p.device) * W)[:, None]
    src = (base + p).reshape(-1)
    held = None if s["lengths"] is None else s["lengths"].reshape(-1)[src]

    def moved(t, to):
        new = t[src]
        if held is None or t.dim() != 4:
            return new
        view = [1, 1, 1, 1]
        view[c["seq_dim"]] = c["positions"]
        keep = torch.arange(c["positions"], device=p.device).view(view) < held.view(-1, 1, 1, 1)
        return torch.where(keep, new, to)

    return [to.copy_(moved(t, to)) for t, to in zip(s["states"], s["out"] or s["states"])]


def _plain_distill(s):
    c = s["case"]
    N, V, T = c["rows"], c["vocab"], c["temp"]
    xs = s["x"].detach()
    x = xs.float()
    ids = s["ids"].to(torch.int64)
    fit = ids >= 0
    at = ids.clamp(min=0)
    lp = s["lp"].double().masked_fill(~fit, NEG)
    if c["tail"] == "drop":
        lp = lp - torch.logsumexp(lp, dim=1, keepdim=True)
    p = torch.exp(lp)
    m = x.amax(1, keepdim=True)
    e = torch.exp((x - m) / T)
    z = e.sum(1, dtype=torch.float64)
    logq = torch.gather(x, 1, at).double() / T - m.double() / T - torch.log(z)[:, None]
    rows = torch.where(fit, p * (lp - logq), 0.0).sum(1)
    factor = torch.ones_like(z)
    if c["tail"] == "bucket":
        rest = (1.0 - p.sum(1)).clamp(min=0.0)
        support = torch.zeros((N, V), device=x.device, dtype=torch.int32).scatter_add_(1, at, fit.to(torch.int32)) > 0
        qt = e.masked_fill(support, 0.0).sum(1, dtype=torch.float64) / z
        there = (rest > 0) & (qt > 0)
        rows = rows + torch.where(there, rest * (torch.log(rest.clamp(min=1e-300)) - torch.log(qt.clamp(min=1e-300))), 0.0)
        factor = torch.where(qt > 0, 1.0 - rest / qt.clamp(min=1e-300), factor)
    w = s["weights"].double() if s["weights"] is not None else torch.ones_like(z)
    rows = torch.where(w != 0, rows * w, 0.0)
    if c["reduction"] == "mean":
        w = w / w.sum()
    loss = rows.float() if c["reduction"] == "none" else rows.sum().float()
    if c["reduction"] == "mean":
        loss = (rows.sum() / (s["weights"].double().sum() if s["weights"] is not None else N)).float()
    if not c["train"]:
        return {"loss": loss}
    if c["reduction"] == "none":
        w = w * s["up"].double()
    q = e / z.float()[:, None]
    if c["tail"] == "bucket":
        grad = torch.where(support, q, q * factor.float()[:, None])
    else:
        grad = q
    grad.scatter_add_(1, at, torch.where(fit, -p, 0.0).float())
    grad *= (w / T).float()[:, None]
    return {"loss": loss, "grad": grad.to(xs.dtype)}


# ---------------------------------------------------------------------------
# the calls
# ---------------------------------------------------------------------------
def _own(s):
    import paged_moe_b200 as pm
    c = s["case"]
    if c["op"] == "top":
        return pm.top_logprobs(s["x"], c["k"], temp=c["temp"], mask=s["mask"], return_lse=True)
    if c["op"] == "select":
        return pm.beam_select(s["x"], s["scores"], n=c["n"], mask=s["mask"], done=s["done"], eos=s["eos"],
                              lengths=s["lengths"], length_penalty=c["penalty"], keep_slots=c["slots"])
    if c["op"] == "reorder":
        # the histories hold one column per token and move whole; the caches move up to their lengths
        n = c["states"]
        dims = [c["seq_dim"] if s["lengths"] is not None else None] * n + [None] * (len(s["states"]) - n)
        return pm.beam_reorder(s["states"], s["parents"], out=s["out"], lengths=s["lengths"], seq_dim=dims)
    loss = pm.distill_loss(s["x"], s["ids"], s["lp"], temp=c["temp"], tail=c["tail"], weights=s["weights"],
                           reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    (grad,) = torch.autograd.grad(loss, s["x"], s["up"] if c["reduction"] == "none" else None)
    return {"loss": loss, "grad": grad}


def run(state):
    if own:
        return _own(state)
    return {"top": _plain_top, "select": _plain_select, "reorder": _plain_reorder,
            "distill": _plain_distill}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _logit_bytes(rows, c):
    size = 4 if c["dtype"] == "f32" else 2
    whole = rows * c["vocab"] * size
    if not c.get("mask"):
        return whole
    # the mask, and the 32-byte sectors that hold an allowed logit
    sectors = rows * c["vocab"] * size / 32.0
    return rows * c["vocab"] / 8.0 + 32.0 * sectors * (1.0 - (1.0 - c["mask"]) ** (32 // size))


def work(case):
    c = case
    if c["op"] == "top":
        return {"bytes": _logit_bytes(c["rows"], c) + c["rows"] * (8 * c["k"] + 4), "flops": 5.0 * c["rows"] * c["vocab"]}
    if c["op"] == "select":
        rows = c["items"] * c["beams"] * (1.0 - c["ended"])
        return {"bytes": _logit_bytes(rows, c) + c["items"] * (17.0 * c["n"] + 9.0 * c["beams"]),
                "flops": 5.0 * rows * c["vocab"]}
    if c["op"] == "reorder":
        rows, W = c["items"] * c["beams"], c["beams"]
        one = c["heads"] * c["positions"] * c["width"] * (4 if c["dtype"] == "f32" else 2) * c["states"]
        one *= (1.0 + c["positions"]) / (2.0 * c["positions"]) if c["ragged"] else 1.0
        one += 4.0 * c["history"]
        if c["in_place"]:  # about half of the rows are written, from the living ones they name
            written, read = 0.5 * (1.0 - 1.0 / W) * rows, 0.33 * rows
        else:  # every row is written; a source is read once however many rows name it
            written, read = rows, rows * (1.0 - (1.0 - 1.0 / W) ** W)
        return {"bytes": one * (written + read) + 4.0 * rows, "flops": 0.0}
    rows = c["rows"] * (0.75 if c["weighted"] else 1.0)
    size = 4 if c["dtype"] == "f32" else 2
    read = rows * (c["vocab"] * size + 8.0 * c["k"])
    return {"bytes": read + (c["rows"] * c["vocab"] * size if c["train"] else 0.0) + 4.0 * c["rows"],
            "flops": (9.0 if c["train"] else 5.0) * rows * c["vocab"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_row(x, words):
    """One row's allowed log-softmax ingredients: (values, log-sum-exp)."""
    v = x.double()
    if words is not None:
        at = torch.arange(v.numel(), device=v.device)
        v = torch.where(((words.to(torch.int64)[at // 32] >> (at % 32)) & 1) == 1, v, NEG)
    return v


def _lse64(v):
    top = v.max()
    return top if top == NEG else top + torch.log(torch.sum(torch.exp(v - top)))


def exact(case, seed):
    c = case
    if c["op"] == "reorder":
        return None  # nothing is computed
    s = prepare(case, seed)
    if c["op"] == "top":
        lps, lses = [], []
        for r in range(c["rows"]):
            v = _exact_row(s["x"][r], None if s["mask"] is None else s["mask"][r]) / c["temp"]
            lse = _lse64(v)
            k = min(c["k"], c["vocab"])
            best = torch.topk(v, k).values
            lp = torch.full((c["k"],), NEG, dtype=torch.float64, device=v.device)
            lp[:k] = torch.where(best > NEG, best - lse, NEG)
            lps.append(lp)
            lses.append(lse)
        return {"ids": None, "logprobs": torch.stack(lps), "lse": torch.stack(lses)}
    if c["op"] == "select":
        B, W, n = c["items"], c["beams"], c["n"]
        scores = []
        for b in range(B):
            totals, ranks, beams = [], [], []
            for w in range(W):
                r = b * W + w
                score, length = float(s["scores"][b, w]), int(s["lengths"][b, w])
                if s["done"] is not None and bool(s["done"][b, w]):
                    t = torch.tensor([score], dtype=torch.float64, device=DEV)
                else:
                    v = _exact_row(s["x"][r], None if s["mask"] is None else s["mask"][r])
                    best = torch.topk(v, min(n, c["vocab"])).values
                    t = score + best[best > NEG] - _lse64(v)
                    length += 1
                totals.append(t)
                ranks.append(t / float(max(length, 1)) ** c["penalty"])
                beams.append(torch.full_like(t, w))
            totals, ranks, beams = torch.cat(totals), torch.cat(ranks), torch.cat(beams)
            at = torch.sort(ranks, descending=True, stable=True).indices[:n]
            row = torch.full((n,), NEG, dtype=torch.float64, device=DEV)
            row[:at.numel()] = totals[at]
            if c["slots"]:
                where, later, placed = {}, [], row.clone()
                for j in range(n):
                    w = int(beams[at[j]]) if j < at.numel() else -1
                    if w >= 0 and w not in where:
                        where[w] = j
                    else:
                        later.append(j)
                for slot in range(n):
                    j = where[slot] if slot in where else later.pop(0)
                    placed[slot] = row[j]
                row = placed
            scores.append(row)
        return {"scores": torch.stack(scores), "parents": None, "tokens": None, "lengths": None, "done": None}
    N, V, T = c["rows"], c["vocab"], c["temp"]
    x, total = s["x"].detach(), torch.zeros((), dtype=torch.float64, device=DEV)
    w = s["weights"].double() if s["weights"] is not None else torch.ones(N, dtype=torch.float64, device=DEV)
    share = w / w.sum() if c["reduction"] == "mean" else w
    losses = []
    grads = torch.empty((N, V), dtype=torch.float64, device=DEV) if c["train"] else None
    back = share * s["up"].double() if c["reduction"] == "none" else share
    for r in range(N):
        ids, lp = s["ids"][r], s["lp"][r].double()
        lp, ids = lp[ids >= 0], ids[ids >= 0].long()
        logq = torch.log_softmax(x[r].double() / T, 0)
        q = torch.exp(logq)
        if c["tail"] == "drop":
            lp = torch.log_softmax(lp, 0)
        p = torch.exp(lp)
        loss = torch.sum(p * (lp - logq[ids]))
        grad = q.clone()
        if c["tail"] == "bucket":
            rest = torch.clamp(1.0 - p.sum(), min=0.0)
            outside = torch.ones(V, dtype=torch.bool, device=DEV)
            outside[ids] = False
            qt = torch.sum(q[outside])
            if float(rest) > 0 and float(qt) > 0:
                loss = loss + rest * (torch.log(rest) - torch.log(qt))
            if float(qt) > 0:
                grad = torch.where(outside, q * (1.0 - rest / qt), grad)
        grad.index_put_((ids,), -p, accumulate=True)
        losses.append(loss * share[r] if float(w[r]) != 0 else total)
        if c["train"]:
            grads[r] = grad * back[r] / T
    losses = torch.stack(losses)
    out = {"loss": losses if c["reduction"] == "none" else losses.sum()}
    if c["train"]:
        out["grad"] = grads
    return out
