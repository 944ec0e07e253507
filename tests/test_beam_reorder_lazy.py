"""beam_reorder moves bytes: a state whose conjugation or sign PyTorch has left
for later goes only into an out of the same kind (no GPU needed)."""

import pytest
import torch

import paged_moe_b200 as pm

_PARENTS = torch.zeros((2, 3), dtype=torch.int32)
_Z = torch.complex(torch.ones(6, 4), torch.ones(6, 4))


@pytest.mark.parametrize("state,out", [
    (_Z.conj(), torch.zeros_like(_Z)), (_Z, torch.zeros_like(_Z).conj()),
    (_Z.conj().imag, torch.zeros(6, 4)[:, :4]), (torch.zeros(6, 4), _Z.conj().imag)])
def test_out_of_another_kind(state, out):
    assert state.is_conj() != out.is_conj() or state.is_neg() != out.is_neg()
    with pytest.raises(ValueError, match="lazily"):
        pm.beam_reorder(state, _PARENTS, out=out)


@pytest.mark.parametrize("state,out", [(_Z.conj(), None), (_Z.conj(), torch.zeros_like(_Z).conj()),
                                       (_Z.conj().resolve_conj(), torch.zeros_like(_Z))])
def test_the_same_kind(state, out):
    with pytest.raises(ValueError, match="CUDA"):  # all that is left to refuse
        pm.beam_reorder(state, _PARENTS, out=out)
