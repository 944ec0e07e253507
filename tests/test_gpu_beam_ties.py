"""top_logprobs of long rows, one CTA each, in which so many elements tie that
the tiles holding them do not fit in its list."""

import numpy as np
import pytest
import torch

import beam_plain as P
import paged_moe_b200 as pm
from test_gpu_beam import DEV, _close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 50, 256])
@pytest.mark.parametrize("share", [None, 0.5])
def test_long_rows_of_ties(share, k, dtype):
    V, repeat, pad = 151937, 30, 1
    rng = np.random.default_rng(80)
    base = np.zeros((6, V))
    base[1] = rng.integers(0, 2, V)
    base[2] = float(torch.finfo(dtype).min)
    base[3, 70000::1000] = 4.0  # fewer than the largest k above the ties
    base[4] = rng.integers(0, 40, V) / 8.0
    base[5, ::2] = -np.inf
    base[5, 1] = -3.0
    base = torch.from_numpy(base).to(dtype)
    x = torch.zeros((6 * repeat, V + pad), dtype=dtype, device=DEV)[:, :V]
    x.copy_(base.to(DEV).repeat(repeat, 1))
    keep, mask = None, None
    if share is not None:
        keep = rng.random((6, V)) < share
        mask = torch.from_numpy(P.pack_bits(keep).view(np.int32)).to(DEV).repeat(repeat, 1)
    got = pm.top_logprobs(x, k, mask=mask, return_lse=True)
    ids, lp, lse = P.top_logprobs(base.double().numpy(), k, 1.0, keep)
    for first in (0, 6 * (repeat - 1)):
        np.testing.assert_array_equal(got["ids"][first:first + 6].cpu().numpy(), ids)
        _close(got["logprobs"][first:first + 6], lp)
        # a row at the lowest value has a log-sum-exp that fp32 holds
        _close(got["lse"][first:first + 6], np.where(np.abs(lse) >= 2.0 ** 128 * (1 - 2.0 ** -25), -np.inf, lse))
    assert torch.equal(got["ids"][:6].repeat(repeat, 1), got["ids"])
