"""beam_reorder carries no derivative: states that have one are refused, as
sources too (no GPU needed)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import paged_moe_b200 as pm

_PARENTS = torch.zeros(1, 3, dtype=torch.int32)


def test_a_source_with_a_gradient():
    leaf = torch.zeros(3, 4, requires_grad=True)
    for source in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="gradient"):
            pm.beam_reorder([source], _PARENTS, out=[torch.zeros(3, 4)])
    with pytest.raises(ValueError, match="gradient"):
        pm.beam_reorder([torch.zeros(3, 2), leaf], _PARENTS, out=[torch.zeros(3, 2), torch.zeros(3, 4)])
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # all that is left to refuse
        pm.beam_reorder([leaf], _PARENTS, out=[torch.zeros(3, 4)])


def test_a_state_with_a_tangent():
    with fwd.dual_level():
        dual = fwd.make_dual(torch.zeros(3, 4), torch.ones(3, 4))
        with pytest.raises(ValueError, match="tangent"):
            pm.beam_reorder([dual], _PARENTS)
        with pytest.raises(ValueError, match="tangent"):
            pm.beam_reorder([dual], _PARENTS, out=[torch.zeros(3, 4)])
        with pytest.raises(ValueError, match="tangent"):
            pm.beam_reorder([torch.zeros(3, 4)], _PARENTS, out=[dual])
