"""The gradients of the objectives element by element, with tolerances in proportion to each element (objectives_rows.py), into
buffers that hold NaN before: no place of a row is left out or wrong, in any of the forms that hold or walk a row."""

import math

import pytest
import torch

from viktor_amd import hip_ops as ops

from . import objectives_rows as rows
from .test_objectives_gpu import FORMS, LONG, lists, policy_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def check(got, want, tol, what):
    bad = rows.outside(got, want, tol)
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError((what, int(bad.sum()), at, float(got[at]), float(want[at]), float(tol[at])))


def fresh(z):
    return torch.full(z.shape, math.nan, dtype=z.dtype, device=DEV)


def sizes(V):
    return (4, 5) if V < 20000 else (2, 3)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", FORMS + LONG)
def test_policy_rows(V, dtype):
    B, T = sizes(V)
    for k, layout in enumerate(("plain", "sliced")):
        z, y, mask, old, ref, g = policy_inputs(B, T, V, dtype, V + k, layout, far=0.1)
        adv = torch.randn((B,) if k else (B, T), generator=g, device=DEV)
        kw = dict(ref_lp=ref, kl_coef=0.05, per="token", inv_n=0.03) if k else dict(eps_hi=0.28)
        want, tol, sound = rows.policy(z, y, mask, old, adv, **kw)
        got = ops.policy_score(z, y, mask, old, adv, **kw, out=fresh(z))["dlogits"]
        assert bool(sound.any())
        check(got[sound], want[sound], tol[sound], layout)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", FORMS + LONG)
def test_preference_rows(V, dtype):
    B, T = (4, 5) if V < 20000 else (2, 2)
    for k, layout in enumerate(("plain", "sliced")):
        z, y, mask, old, ref, g = policy_inputs(B, T, V, dtype, V + k, layout)
        mask[1, :1] = True
        kw = dict(beta=0.3) if k else dict(pairs=torch.tensor([[1, 0], [0, B - 1], [1, 0]], device=DEV), smoothing=0.1,
                                           lengths=1 + torch.rand(B, generator=g, device=DEV))
        want, tol, margin, mtol = rows.preference(z, y, mask, ref, **kw)
        got = ops.preference_score(z, y, mask, ref, **kw, out=fresh(z))
        check(got["margin"], margin, mtol, layout)
        check(got["dlogits"], want, tol, layout)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", FORMS + LONG)
def test_distill_rows(V, dtype):
    B, T = sizes(V)
    for k, layout in enumerate(("plain", "sliced")):
        tau = (1.0, 1.7)[k]
        z, y, mask, _, _, g = policy_inputs(B, T, V, dtype, V + k, layout)
        val, ids, lse = lists(z, min(V, (24, 128)[k]), g, (F32, BF16)[k], torch.int32, tau)
        if V > 7:
            ids[0, 0, 1] = ids[0, 0, 0]
            ids[0, 1, 2], ids[0, 2, 3] = -1, V
        w = torch.where(mask, 0.2 + torch.rand(B, T, generator=g, device=DEV), 0.0)
        for kw in (dict(weights=w), dict(t_lse=lse, inv_n=0.1)):
            want, tol, kl, ktol = rows.distill(z, val, ids, temperature=tau, **kw)
            got = ops.distill_score(z, val, ids, temperature=tau, **kw, out=fresh(z))
            check(got["kl"], kl, ktol, layout)
            check(got["dlogits"], want, tol, layout)
