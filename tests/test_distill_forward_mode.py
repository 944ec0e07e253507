"""A dual tensor's derivative is refused instead of dropped (no GPU needed)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import paged_moe_b200 as pm

_REST = (torch.zeros((3, 5), dtype=torch.int32), torch.zeros((3, 5)))


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(requires_grad, reduction):
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros((3, 100), requires_grad=requires_grad), torch.ones(3, 100))
        with pytest.raises(ValueError, match="forward-mode"):
            pm.distill_loss(x, *_REST, reduction=reduction)
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            pm.distill_loss(x, *_REST, reduction=reduction)
        with pytest.raises(ValueError, match="CUDA"):  # the primal alone: all that is left to refuse
            pm.distill_loss(fwd.unpack_dual(x).primal.detach(), *_REST, reduction=reduction)
    with pytest.raises(ValueError, match="CUDA"):
        pm.distill_loss(x.detach(), *_REST, reduction=reduction)
