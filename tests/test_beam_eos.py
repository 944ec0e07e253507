"""beam_select's eos is a token id or None (no GPU needed)."""

import pytest
import torch

import paged_moe_b200 as pm


@pytest.mark.parametrize("eos", [-1, -2, 1 << 31])
def test_eos_that_is_no_token(eos):
    """-1 stood for None inside, and "done" came back as None."""
    with pytest.raises(ValueError, match="eos"):
        pm.beam_select(torch.zeros((2, 3, 100)), torch.zeros((2, 3)), eos=eos)


def test_none_and_tokens():
    for eos in (None, 0, 99):
        with pytest.raises(ValueError, match="CUDA"):  # all that is left to refuse
            pm.beam_select(torch.zeros((2, 3, 100)), torch.zeros((2, 3)), eos=eos)
