"""The tolerances of tests/objectives_rows.py hold what they should and reject gradients with a place left out (no GPU)."""

import math

import pytest
import torch

from . import objectives_rows as rows

SIZES = [1, 2, 7, 8, 13, 16, 33, 127, 343, 385, 500, 1367, 1537, 2500, 5463, 8191, 12289, 21847, 22600, 45100, 60001, 87383,
         90200, 180300, 250001]


def _inputs(B, T, V, dtype):
    g = torch.Generator().manual_seed(V)
    y = torch.randint(0, V, (B, T), generator=g)
    z = 2 * torch.randn(B, T, V, generator=g)
    z.scatter_add_(2, y[..., None], math.log(V) + 3 * torch.rand(B, T, 1, generator=g))
    z = z.to(dtype)
    lp = torch.log_softmax(z.double(), -1).gather(2, y[..., None])[..., 0].float()
    return z, y, torch.ones(B, T, dtype=torch.bool), lp, g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", SIZES)
def test_a_place_left_out_is_rejected(V, dtype):
    """The definition's own gradient, rounded, is accepted; with its last element, its first, or 16 bytes anywhere at zero it is
    not, wherever the token has a gradient."""
    B, T = 2, 2
    z, y, mask, lp, g = _inputs(B, T, V, dtype)
    old = lp + 0.05 * torch.randn(B, T, generator=g)
    ref = lp + 0.3 * torch.randn(B, T, generator=g)
    val, ids = torch.topk(z.float() + 0.7 * torch.randn(B, T, V, generator=g), min(V, 24), -1)
    adv = torch.tensor([1.0, -2.0])
    leaf = z.double().requires_grad_(True)
    logp = torch.log_softmax(leaf, -1)
    lp64 = logp.gather(2, y[..., None])[..., 0]
    r, a = torch.exp(lp64 - old.double()), adv.double()[:, None]
    x = ref.double() - lp64
    loss = ((-torch.minimum(r * a, r.clamp(0.8, 1.2) * a) + 0.05 * (torch.exp(x) - x - 1)).mean(1)).mean()
    s = (lp64 - ref.double()).sum(1)
    pair = -torch.nn.functional.logsigmoid(0.3 * (s[0] - s[1]))
    log_q = torch.log_softmax(val.double(), -1)
    kl = (log_q.exp() * (log_q - logp.gather(2, ids))).sum(-1).mean()
    for want, tol, loss in ((*rows.policy(z, y, mask, old, adv, ref, kl_coef=0.05)[:2], loss),
                            (*rows.preference(z, y, mask, ref, beta=0.3)[:2], pair), (*rows.distill(z, val, ids)[:2], kl)):
        # autograd's c onehot - c p cancels in 64 bits where p is next to 1
        grad = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
        assert bool(((grad - want).abs() <= 1e-12 * want.abs().amax() + 1e-12 * want.abs()).all())
        got = want.to(dtype)
        assert not bool(rows.outside(got, want, tol).any())
        if V == 1:
            continue
        live = want[..., 0].abs() > 0
        assert bool(live.any())
        n = 16 // got.element_size()
        for lo, hi in [(V - 1, V), (0, 1)] + [(int(i), int(i) + n) for i in torch.randint(0, V, (20,), generator=g)]:
            bad = got.clone()
            bad[..., lo:hi] = 0
            assert bool(rows.outside(bad, want, tol)[..., lo:hi].flatten(2).any(-1)[live].all()), (lo, hi)
            bad[..., lo:hi] = math.nan
            assert bool(rows.outside(bad, want, tol)[..., lo:hi].all())
        assert bool(rows.outside(got * 1.02, want, tol)[live].any())
