"""The objectives as the training paths call them: the token objective of gspo_update, pairs, distillation from a teacher."""

import pytest
import torch

from viktor_amd import gspo, hip_ops as ops, objectives, train as TR
from viktor_amd.synthetic import make_model

from . import objectives_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(seed, k=1):
    """Three windows of three calls (window 1 with equal rewards), frames and prefix lengths."""
    g = torch.Generator().manual_seed(seed)
    G, P = 3, 40
    fr = torch.randn(3, P, 512, generator=g).to(DEV)
    plens = torch.tensor([40, 31, 17], device=DEV)
    calls = ["".join("ACGT"[int(i)] for i in torch.randint(0, 4, (int(n),), generator=g))
             for n in torch.randint(3, 60, (3 * G,), generator=g)]
    ended = [True] * 4 + [False] + [True] * 4
    reward = [[0.9, 0.5, 0.7], [0.4, 0.4, 0.4], [0.2, 0.8, 0.3]]
    return fr, plens, calls, ended, reward, G


@pytest.mark.parametrize("k", [1, 4])
def test_token_objective_is_the_loop_of_its_parts(k):
    """gspo_update with the token objective and a KL term, two steps: the weights of a loop of train_logits,
    token_policy_loss, backward and the optimiser, bit for bit; the statistics at a first step, where the policy is its own
    old one."""
    fr, plens, calls, ended, reward, G = _inputs(5)
    make = lambda seed: make_model(k, n_layers=2, seed=seed, norm_jitter=0.1).to(DEV)  # noqa: E731
    m1, m2, ref = make(62), make(62), make(63)
    o1, o2 = (TR.HipAdamW(list(m.parameters()), lr=1e-4) for m in (m1, m2))
    kw = dict(eps=0.2, eps_hi=0.3, objective="token", ref_model=ref, kl_coef=0.05)
    st = TR.gspo_update(m1, o1, fr, plens, calls, ended, reward, G, updates=1, micro=3, **kw)
    adv, live = gspo.advantages(torch.tensor(reward, dtype=torch.float64).numpy(), std_floor=0.003)
    seqs = [(b, j) for b in live for j in range(G)]
    o2.zero_grad()
    want = {"pg": 0.0, "kl": 0.0}
    for i in range(0, len(seqs), 3):
        mb = seqs[i:i + 3]
        ix = torch.tensor([b for b, _ in mb], device=DEV)
        args = (fr[ix], plens[ix], [calls[b * G + j] for b, j in mb], [ended[b * G + j] for b, j in mb])
        z, y, mask = TR.token_logprobs_train(m2, *args, group_size=G)
        with torch.no_grad():
            zr = TR.token_logprobs_train(ref, *args, group_size=G)[0]
        zero = torch.zeros(y.shape, device=DEV)
        old, ref_lp = (ops.policy_score(t.detach(), y, mask, zero, zero, grad=False)["lp"] for t in (z, zr))
        a = torch.tensor([adv[b, j] for b, j in mb], device=DEV, dtype=torch.float32)
        loss, pg, kl, lp = objectives.token_policy_loss(z, y, mask, old, a, ref_lp, 0.2, 0.3, 0.05, inv_n=1.0 / len(seqs))
        loss.backward()
        # the formula in 64 bits on the same logits: each value off by a few 32-bit roundings of terms of size 10
        _, exact = plain.policy(z.detach(), y, mask, old, a, ref_lp, 0.2, 0.3, 0.05, inv_n=1.0 / len(seqs))
        assert abs(float(loss.detach()) - float(exact["loss"].detach())) < 1e-5
        want["pg"] += float((pg.sum(1) / mask.sum(1)).sum())
        want["kl"] += float((kl.sum(1) / mask.sum(1)).sum())
    o2.step()
    assert all(torch.equal(p, q) for p, q in zip(m1.parameters(), m2.parameters()))
    assert st["n"] == len(seqs) == 6 and st["clip"] == 0 and st["ratio"] < 6 * 2e-6 and st["kl"] > 0
    assert abs(st["pg"] - want["pg"]) < 1e-5 and abs(st["kl"] - want["kl"]) < 1e-4 * want["kl"]
    st = TR.gspo_update(m1, o1, fr, plens, calls, ended, reward, G, updates=2, micro=3, **kw)
    assert len(st["grad_norm"]) == 2 and st["grad_norm"][0] > 0


def test_sequence_objective_keeps_its_bits():
    """The new arguments left at their defaults change nothing."""
    fr, plens, calls, ended, reward, G = _inputs(6)
    out = []
    for kw in ({}, {"objective": "sequence", "eps_hi": 0.2, "kl_coef": 0.0}):
        m = make_model(1, n_layers=1, seed=64).to(DEV)
        opt = TR.HipAdamW(list(m.parameters()), lr=1e-4)
        st = TR.gspo_update(m, opt, fr, plens, calls, ended, reward, G, updates=1, micro=3, eps=0.2, **kw)
        assert "kl" not in st
        out.append([p.detach().clone() for p in m.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_update_refuses():
    fr, plens, calls, ended, reward, G = _inputs(7)
    m = make_model(1, n_layers=1, seed=65).to(DEV)
    for kw in ({"objective": "batch"}, {"kl_coef": 0.1}, {"ref_model": m}, {"objective": "token", "kl_coef": 0.1}):
        with pytest.raises(ValueError):
            TR.gspo_update(m, None, fr, plens, calls, ended, reward, G, **kw)


@pytest.mark.parametrize("k", [1, 4])
def test_pairs_of_calls(k):
    """The best and the worst call of each window, through the model: value and gradient by the logits as the formula gives
    them in 64 bits; a step against the gradient raises the margin."""
    fr, plens, calls, ended, reward, G = _inputs(8)
    m = make_model(k, n_layers=2, seed=66, norm_jitter=0.1).to(DEV)
    ix = torch.arange(3, device=DEV).repeat_interleave(G)
    args = (fr[ix], plens[ix], calls, ended)
    ref_lp, mask = gspo.token_logprobs(m, *args)
    pairs = torch.tensor([[0, 1], [7, 6], [7, 8]], device=DEV)
    loss, margin, lp = TR.pair_loss(m, *args, ref_lp=ref_lp, pairs=pairs, beta=0.2, group_size=G)
    # the same model: both sides' ratios are 1 up to the 32-bit log-probabilities of the reference, 2e-6 a token of 60
    assert float(margin.abs().max()) < 0.2 * 2 * 60 * 2e-6
    assert abs(float(loss.detach()) - 0.6931472) < 0.2 * 60 * 2e-6 + 1e-6
    loss.backward()
    grads = [p.grad.clone() for p in m.parameters() if p.grad is not None]
    assert all(bool(torch.isfinite(g).all()) for g in grads) and sum(float(g.norm()) for g in grads) > 0
    z, y, _ = TR.token_logprobs_train(m, *args, group_size=G)
    got = torch.autograd.grad(objectives.preference_loss(z, y, mask, ref_lp, pairs, 0.2)[0], z)[0]
    leaf, want = plain.preference(z.detach(), y, mask, ref_lp, pairs, 0.2)
    want = torch.autograd.grad(want["loss"], leaf)[0]
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * want.abs().max()).all())
    with torch.no_grad():
        scale = 0.05 / sum(float(g.norm()) ** 2 for g in grads) ** 0.5
        for p in m.parameters():
            if p.grad is not None:
                p -= scale * p.grad
    again = TR.pair_loss(m, *args, ref_lp=ref_lp, pairs=pairs, beta=0.2, group_size=G)[0]
    assert float(again.detach()) < float(loss.detach())


@pytest.mark.parametrize("k,renormalise", [(1, False), (4, False), (4, True)])
def test_distillation_from_a_teacher(k, renormalise):
    """A teacher's lists through the student's loss: nothing to learn from itself, the formula's value and gradient from
    another teacher, PAD and weightless bases left out."""
    fr, plens, calls, ended, reward, G = _inputs(9)
    seqs = calls[:3]
    weights = [torch.rand(len(s), generator=torch.Generator().manual_seed(i)).numpy() for i, s in enumerate(seqs)]
    weights[1][:8] = 0
    teacher, student = (make_model(k, n_layers=1, seed=s, norm_jitter=0.1).to(DEV) for s in (67, 68))
    n = min(teacher.cfg.vocab_size, 24)
    own = gspo.teacher_lists(student, fr, plens, seqs, n, 1.5)
    if k == 1:  # the whole vocabulary in the list; the two forwards give the same logits
        loss, kl = TR.distill_frame_loss(student, fr, seqs, own, weights, plens, 1.5)
        assert float(kl.abs().max()) < 1e-5 and abs(float(loss.detach())) < 1e-5
    lists = gspo.teacher_lists(teacher, fr, plens, seqs, n, 1.5)
    loss, kl = TR.distill_frame_loss(student, fr, seqs, lists, weights, plens, 1.5, renormalise)
    loss.backward()
    grads = [p.grad for p in student.parameters() if p.grad is not None]
    assert float(loss.detach()) > 0 and all(bool(torch.isfinite(g).all()) for g in grads) and sum(float(g.norm()) for g in grads) > 0
    tokens_in, targets, w = student.batch(seqs, weights)
    z = TR.train_logits(student, fr, tokens_in, plens)
    w = (w * (targets != 0)).to(DEV)
    leaf, want = plain.distill(z.detach(), *lists[:2], None if renormalise else lists[2], w, 1.5)
    assert abs(float(loss.detach()) - float(want["loss"].detach())) < 2e-5 * max(1.0, float(want["loss"].detach()))
    assert bool((kl[~(w > 0)] == 0).all())
    got = torch.autograd.grad(objectives.distill_loss(z, *lists[:2], None if renormalise else lists[2], w, 1.5)[0], z)[0]
    want = torch.autograd.grad(want["loss"], leaf)[0]
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * want.abs().max()).all())
