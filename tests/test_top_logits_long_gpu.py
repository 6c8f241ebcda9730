"""The log-sum-exp of top_logits over long rows."""

import math

import pytest
import torch

from viktor_amd import hip_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("V", [200003, 2 ** 22 + 5, 2 ** 24 + 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_top_log_sum_exp_of_very_long_rows(V, dtype):
    """One logit above millions of equal ones: no rounding that each addition makes to the same side. The exponential is off by
    2^-24 |z - top| of itself with the product and the difference each and by its ulp, 2^-23; the sum in 64 bits by nothing; the
    result by half its last place."""
    z = torch.full((2, V), -1.0, dtype=dtype, device=DEV)
    z[0, V // 3], z[1, V - 1], z[1, 0] = 0.0, 1.5, 1.25
    for tau in (1.0, 0.5):
        values, ids, lse = ops.top_logits(z, 1, tau)
        want = torch.logsumexp(z.double() / tau, -1)
        off = 2.0 ** -24 * (2 * 2.5 / tau + 2) + 2.0 ** -24 * want.abs()
        assert ids[:, 0].tolist() == [V // 3, V - 1] and values[:, 0].tolist() == [0.0, 1.5]
        assert bool(((lse.double() - want).abs() <= off).all()), (lse.double() - want).tolist()


@pytest.mark.parametrize("V", [343, 5463, 21847, 87383, 180000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_top_log_sum_exp_of_equal_logits(V, dtype):
    """Rows in registers: 2^-24 more with each addition, eight of a vector, 22 vectors of a thread and ten between threads."""
    z = torch.full((2, V), -1.0, dtype=dtype, device=DEV)
    z[0, V // 3], z[1, V - 1], z[1, 0] = 0.0, 1.5, 1.25
    for tau in (1.0, 0.5):
        lse = ops.top_logits(z, 1, tau)[2]
        want = torch.logsumexp(z.double() / tau, -1)
        off = 2.0 ** -24 * (2 * 2.5 / tau + 2 + 40) + 2.0 ** -24 * want.abs()
        assert bool(((lse.double() - want).abs() <= off).all()), (lse.double() - want).tolist()
