"""The objectives on logits in 64 bits, from their definitions, with autograd for the gradients; and how far 32-bit kernels
may be from them."""

import math

import torch


def counting(targets, mask, V):
    return mask.bool() & (targets >= 0) & (targets < V)


def _tokens(logits, targets, mask):
    """(leaf, log-probabilities with zeros where a token does not count, which count); rows that do not count are zeroed
    before anything is computed, whatever they hold."""
    V = logits.shape[2]
    on = counting(targets, mask, V)
    z = torch.where(on[..., None], logits.double(), 0.0).requires_grad_(True)
    lp = torch.log_softmax(z, -1).gather(2, targets.clamp(0, V - 1)[..., None])[..., 0]
    return z, torch.where(on, lp, 0.0), on


def policy(logits, targets, mask, old_lp, adv, ref_lp=None, eps_lo=0.2, eps_hi=0.2, kl_coef=0.0, per="sequence", inv_n=None):
    z, lp, on = _tokens(logits, targets, mask)
    B = logits.shape[0]
    r = torch.exp(lp - torch.where(on, old_lp.double(), 0.0))
    a = adv.double()[:, None] if adv.dim() == 1 else adv.double()
    a = torch.where(on, a.expand_as(lp), 0.0)
    pg = -torch.minimum(r * a, r.clamp(1 - eps_lo, 1 + eps_hi) * a)
    kl, term = None, pg
    if ref_lp is not None:
        x = torch.where(on, ref_lp.double(), 0.0) - lp
        kl = torch.where(on, torch.exp(x) - x - 1, 0.0)
        term = pg + kl_coef * kl
    n = on.double()
    if per == "sequence":
        w = (1.0 / max(B, 1) if inv_n is None else inv_n) * n / n.sum(1, keepdim=True).clamp(min=1)
    else:
        w = n / n.sum().clamp(min=1) if inv_n is None else inv_n * n
    loss = (w * torch.where(on, term, 0.0)).sum()
    return z, {"loss": loss, "pg": torch.where(on, pg, 0.0), "kl": kl, "lp": lp}


def preference(logits, targets, mask, ref_lp=None, pairs=None, beta=0.1, target=0.0, smoothing=0.0, lengths=None, inv_n=None):
    z, lp, on = _tokens(logits, targets, mask)
    B = logits.shape[0]
    s = (lp - (0.0 if ref_lp is None else torch.where(on, ref_lp.double(), 0.0))).sum(1)
    if lengths is not None:
        s = s / lengths.double()
    if pairs is None:
        pairs = torch.arange(B, device=logits.device).view(-1, 2)
    P = pairs.shape[0]
    good = ((pairs >= 0) & (pairs < B)).all(1)
    c, r = pairs.clamp(0, max(B - 1, 0)).unbind(1)
    h = torch.where(good, beta * (s[c] - s[r]) - target, 0.0)
    ls = torch.nn.functional.logsigmoid
    each = -(1 - smoothing) * ls(h) - smoothing * ls(-h)
    loss = (1.0 / max(P, 1) if inv_n is None else inv_n) * torch.where(good, each, 0.0).sum()
    return z, {"loss": loss, "margin": h, "lp": lp}


def distill(logits, values, ids, t_lse=None, weights=None, temperature=1.0, inv_n=None):
    B, T, V = logits.shape
    w = torch.ones(B, T, dtype=torch.float64, device=logits.device) if weights is None else weights.double()
    on = w > 0
    z = torch.where(on[..., None], logits.double(), 0.0).requires_grad_(True)
    logp = torch.log_softmax(z / temperature, -1)
    there = on[..., None] & (ids >= 0) & (ids < V) & (values > -math.inf)
    t = torch.where(there, values.double() / temperature, -1e5)
    some = there.any(-1, keepdim=True)
    log_q = torch.log_softmax(t, -1) if t_lse is None else t - torch.where(on, t_lse.double(), 0.0)[..., None]
    q = torch.where(there & some, log_q.exp(), 0.0)
    kl = torch.where(there, q * (log_q - logp.gather(2, ids.long().clamp(0, V - 1))), 0.0).sum(-1)
    w = torch.where(on, w, 0.0)
    if inv_n is None:
        w = w / w.sum() if bool(w.sum() > 0) else w
    else:
        w = w * inv_n
    return z, {"loss": temperature ** 2 * (w * kl).sum(), "kl": kl}


def lp_tolerance(logits, V, tau=1.0):
    """How far lp may be off. A term exp(t), t = (z - max) / tau: t is off by two roundings and the scale's (3 2^-24 |t|),
    the exponential by an ulp (2^-23); over a softmax the mean of -t is at most log V. Adding n terms one after the other
    (100 a thread at most where rows stay in registers, V / 1024 a thread past that) and 16 partial sums: 2^-24 each, all to
    one side at worst. The logarithm: 2^-24; lp itself: half a step of its largest size, and of the difference under it."""
    fin = logits.double()[torch.isfinite(logits)]
    far = float((fin.max() - fin.min()) / tau) if fin.numel() else 0.0
    u = 2.0 ** -24
    return u * (3 * math.log(V) + 2 + min(V, 100 + V / 1024) + 16 + 1 + 3 * (far + math.log(V)))


def gradient_tolerance(want, coef, dtype, lp_tol):
    """|got - want| allowed per element: want = c (onehot - p): p's error relative to p is lp's and its own exponential's,
    c's is a few roundings; then half a step of the type."""
    half = torch.finfo(dtype).eps / 2
    return (2 * lp_tol + 2.0 ** -20) * coef + half * want.abs() + 1e-37
