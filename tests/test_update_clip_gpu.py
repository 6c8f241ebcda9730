"""The borders of the clip in gspo_update: what it counts by them, and their defaults."""

import pytest
import torch

from viktor_amd import train as TR
from viktor_amd.synthetic import make_model

from .test_objectives_paths_gpu import _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("eps,eps_hi,each", [(0.2, 0.3, 1), (0.4, 0.1, 1), (0.2, None, 2), (0.4, 0.3, 0)])
def test_sequence_objective_counts_what_its_borders_clip(eps, eps_hi, each, monkeypatch):
    """Ratios of 0.7, 1 and 1.25 in each window: those under 1 - eps or over 1 + eps_hi are the clipped ones."""
    fr, plens, calls, ended, reward, G = _inputs(10)
    real = TR.sequence_ratio_loss

    def moved(*args):
        loss, s, pg, lp = real(*args)
        return loss, torch.tensor([0.7, 1.0, 1.25], device=DEV), pg, lp

    monkeypatch.setattr(TR, "sequence_ratio_loss", moved)
    m = make_model(1, n_layers=1, seed=70).to(DEV)
    opt = TR.HipAdamW(list(m.parameters()), lr=1e-4)
    kw = {} if eps_hi is None else {"eps_hi": eps_hi}
    st = TR.gspo_update(m, opt, fr, plens, calls, ended, reward, G, updates=1, micro=3, eps=eps, **kw)
    assert st["n"] == 6 and st["clip"] == 2 * each


@pytest.mark.parametrize("kw,want", [({}, 4e-4), ({"objective": "token"}, 0.2), ({"objective": "token", "eps": 0.1}, 0.1),
                                     ({"eps": 0.1}, 0.1)])
def test_clip_by_default(kw, want, monkeypatch):
    """A sequence's ratio is a mean over its length, a token's is not: each objective's clip is its own by default."""
    fr, plens, calls, ended, reward, G = _inputs(11)
    seen = []
    for name, at in (("sequence_ratio_loss", 6), ("token_policy_loss", 6)):
        real = getattr(TR, name)
        monkeypatch.setattr(TR, name, lambda *args, _real=real, _at=at, **more: (seen.append(args[_at:_at + 2]),
                                                                                 _real(*args, **more))[1])
    m = make_model(1, n_layers=1, seed=71).to(DEV)
    TR.gspo_update(m, TR.HipAdamW(list(m.parameters()), lr=1e-4), fr, plens, calls, ended, reward, G, updates=1, micro=3, **kw)
    assert seen and all(s == (want, want) for s in seen)
