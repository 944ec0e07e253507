"""beam_reorder on states whose rows are windows over the same memory: moved in
place, or written, they would race (no GPU needed)."""

import pytest
import torch

import paged_moe_b200 as pm

_PARENTS = torch.zeros((2, 3), dtype=torch.int32)
_LENGTHS = torch.ones((2, 3), dtype=torch.int32)


def _strided(sizes, strides):
    return torch.zeros(sum((n - 1) * s for n, s in zip(sizes, strides)) + 1).as_strided(sizes, strides)


@pytest.mark.parametrize("sizes,strides,kw", [
    ((6, 10), (2, 1), {}),               # rows
    ((6, 3, 4), (12, 3, 1), {}),         # runs of a row
    ((6, 3, 4), (4, 16, 1), {}),         # rows inside the runs
    ((6, 2, 5, 4), (40, 19, 4, 1), dict(seq_dim=2, lengths=_LENGTHS)),
    ((6, 5), (3, 1), dict(seq_dim=1, lengths=_LENGTHS)),
])
def test_windows_are_refused(sizes, strides, kw):
    state = _strided(sizes, strides)
    with pytest.raises(ValueError, match="windows"):
        pm.beam_reorder(state, _PARENTS, **kw)
    with pytest.raises(ValueError, match="windows"):
        pm.beam_reorder(torch.zeros(sizes), _PARENTS, out=state, **kw)


@pytest.mark.parametrize("sizes,strides", [
    ((6, 10), (10, 1)), ((6, 10), (13, 1)), ((6, 3, 4), (4, 24, 1)), ((6, 3, 4), (5, 31, 1)), ((6, 3, 4), (40, 9, 1)),
    ((6, 1, 4), (4, 1, 1)), ((6,), (7,)), ((6, 1), (1, 1)), ((6, 0), (1, 1)),
])
def test_rows_apart_are_not(sizes, strides):
    with pytest.raises(ValueError, match="CUDA"):  # all that is left to refuse
        pm.beam_reorder(_strided(sizes, strides) if 0 not in sizes else torch.zeros(sizes), _PARENTS)
