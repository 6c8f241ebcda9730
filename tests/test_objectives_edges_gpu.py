"""The type's lowest value as a mask, in the objectives' logits and lists: what the definitions give in 64 bits."""

import math

import pytest
import torch

from viktor_amd import hip_ops as ops

from . import objectives_rows as rows
from .test_objectives_gpu import lists, policy_inputs
from .test_objectives_rows_gpu import check, fresh

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def check_distill(z, val, ids, **kw):
    want, tol, kl, ktol = rows.distill(z, val, ids, **kw)
    got = ops.distill_score(z, val, ids, **kw, out=fresh(z))
    check(got["kl"], kl, ktol, "kl")
    check(got["dlogits"], want, tol, "gradient")
    w = torch.ones_like(kl) if kw.get("weights") is None else kw["weights"].double()
    w = w / w.sum() if kw.get("inv_n") is None else w * kw["inv_n"]
    scale = kw.get("temperature", 1.0) ** 2
    check(got["loss"], scale * (w * kl).sum(), scale * ((w * ktol).sum() + 2 * rows.U * (w * kl).sum().abs()), "loss")


@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0])
@pytest.mark.parametrize("vdtype", [BF16, F32])
@pytest.mark.parametrize("V", [7, 343, 5463, 25000, 190000])
def test_distill_lists_that_end_in_the_lowest_value(V, vdtype, tau):
    """A teacher whose mask writes the type's lowest value leaves it in its lists: a weight of 0, at every temperature, also
    where the value over the temperature is beyond 32 bits."""
    z, _, _, _, _, g = policy_inputs(2, 3, V, (F32, BF16)[V % 2], V)
    K = min(V, 24)
    val, ids, _ = lists(z, K, g, vdtype, torch.int32)
    val[..., 3:] = torch.finfo(vdtype).min
    val[1, 0, 1:] = torch.finfo(vdtype).min
    lse = (val.double() / tau).logsumexp(-1).float() + 0.1
    check_distill(z, val, ids, temperature=tau)
    check_distill(z, val, ids, temperature=tau, t_lse=lse, inv_n=0.2)
    # its own lists, as top_logits gives them
    t = torch.full((2, 3, V), torch.finfo(vdtype).min, dtype=vdtype, device=DEV)
    t[..., 1:4] = torch.randn(2, 3, 3, generator=g, device=DEV).to(vdtype)
    val, ids, lse = ops.top_logits(t, K, tau)
    check_distill(z, val, ids, temperature=tau)
    check_distill(z, val, ids, temperature=tau, t_lse=lse)


@pytest.mark.parametrize("tau", [0.7, 1.0, 2.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [7, 343, 5463, 25000, 190000])
def test_distill_rows_of_the_lowest_value(V, dtype, tau):
    """A row whose mask leaves nothing, written as the type's lowest value, is a uniform one: of the student, of the list, of
    both. So is a row of one far value, and one of a large common size keeps its differences."""
    z, _, _, _, _, g = policy_inputs(2, 5, V, dtype, V)
    K = min(V, 16)
    val, ids, lse = lists(z, K, g, dtype, torch.int32, tau)
    low = torch.finfo(dtype).min
    z[0, 0], z[0, 1], z[0, 2] = low, 1e30, -1e37
    z[1, 0] = low
    z[1, 1] = 2.0 ** 20 + 8192 * torch.randint(0, 2, (V,), generator=g, device=DEV)  # (in either type without a rounding)
    z[1, 2] = low
    z[1, 2, ids[1, 2].long()] = 1.0  # (what the list does not name is masked)
    val[1, 0] = low
    val[1, 3] = low
    val[1, 4] = -1e33
    check_distill(z, val, ids, temperature=tau)
    lse[1, 0], lse[1, 3], lse[1, 4] = 5.0, 6.0, 7.0  # (no weight at all against a teacher's sum)
    check_distill(z, val, ids, temperature=tau, t_lse=lse, inv_n=0.1)
