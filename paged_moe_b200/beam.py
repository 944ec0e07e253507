"""Beam search on the device: the selection over beams and vocabulary, and
the reordering of the states that belong to the beams.

The reference decodes one sequence per request (pagedmoe/verify_decode.py:727
generate_step); this is the step that keeps several.  It reads the logits
after each beam, as `sample_rows` does, and leaves scores, parents and tokens
on the device: a whole step runs without the host.
"""

from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from . import _lib as L


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: Optional[int] = None,
                mask: Optional[torch.Tensor] = None, done: Optional[torch.Tensor] = None, eos: Optional[int] = None,
                lengths: Optional[torch.Tensor] = None, length_penalty: float = 0.0, keep_slots: bool = False):
    """The n best continuations of every item over its beams and the vocabulary.

    logits [B, W, V] (or [B*W, V]) fp32 or bf16: row w of item b follows beam
    w (processors, where wanted, run before: apply_processors).  scores [B, W]
    fp32: log-probability of each beam so far, -inf for a beam that is not
    there (at the first step all but one).  n: candidates per item, 2 W when
    not given.  mask: packed allowed-token words, [B*W, words] or [words].
    eos: the token that ends a beam.  done [B, W] bool: beams that have ended;
    they offer themselves once, with token eos, score and length unchanged,
    and their logits are not read.  lengths [B, W] int32: tokens of each beam
    so far.

    Candidates are ranked by (score + logit - row log-sum-exp) in 64 bits,
    divided by length ** length_penalty with the new token counted; ties go
    to the lower beam, then the larger logit, then the lower token.
    keep_slots (n == W): the best child of every beam that lives on takes its
    parent's place, the others fill the free places; beam_reorder in place
    then moves only the beams that ended.

    Returns {"scores" [B, n] fp32 (not divided), "parents" [B, n] int32 (beam
    of the item), "tokens" [B, n] int32}, with "lengths" when lengths are
    given and "done" [B, n] bool when eos is.  Places without a candidate
    hold -inf, -1, -1, length 0.  W <= 64, n <= 256.
    """
    if eos is not None and eos < 0:  # -1 is how the library is told that there is none
        raise ValueError("eos must be a token id, None without one")
    if n is None:
        n = scores.shape[-1] if keep_slots else 2 * scores.shape[-1]
    out = L.ext().beam_select(logits, scores, n, mask, done, -1 if eos is None else eos, lengths, length_penalty,
                              keep_slots)
    res = {"scores": out[0], "parents": out[1], "tokens": out[2]}
    if lengths is not None:
        res["lengths"] = out[3]
    if eos is not None:
        res["done"] = out[4]
    return res


def beam_reorder(states: Union[torch.Tensor, Sequence[torch.Tensor]], parents: torch.Tensor,
                 out: Union[torch.Tensor, Sequence[torch.Tensor], None] = None,
                 lengths: Optional[torch.Tensor] = None,
                 seq_dim: Union[int, None, Sequence[Optional[int]]] = None):
    """Moves every state's rows to the beams that continue them.

    states: one tensor or several of any type, [B*W, ...] with the beams of an
    item next to one another (key-value caches, recurrent states, token
    histories).  parents [B, W] int32, as beam_select gives them (a slice
    [:, :W] of more candidates will do): row b*W + j takes what row b*W +
    parents[b, j] held before the call.  A parent outside [0, W) leaves the
    row its own.

    Without out the states are reordered in place, and only rows whose parent
    is another row are touched.  With out (one tensor per state, the same
    shapes; a double buffer) every row is written there and the states stay.

    lengths [B, W] or [B*W] int32 (those before the reorder) with seq_dim, the
    dimension of a state that counts positions (one for all states, or one
    per state, None for a state without): only the first lengths[parent] positions
    move; positions behind them stay as they were.

    A state has to be dense from its position dimension on (without
    positions: any split into leading dimensions that collapse and a dense
    rest), and its rows must not overlap, nor states, out, parents and lengths
    one another.  All states move in one launch (up to 128).  No derivative is carried: where autograd is
    on, states and outs that require a gradient are refused, and dual tensors
    always.  Returns out, or the states.
    """
    one = isinstance(states, torch.Tensor)
    s = [states] if one else list(states)
    o = None if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    dims = seq_dim if isinstance(seq_dim, (list, tuple)) else [seq_dim] * len(s)
    flat = [-1 if d is None else d + t.dim() if d < 0 else d for d, t in zip(dims, s)] if len(dims) == len(s) else []
    if any(d is not None and f < 0 for d, f in zip(dims, flat)):
        raise ValueError("seq_dim is out of range")
    L.ext().beam_reorder(s, parents, o, lengths, flat)
    return states if out is None else out
