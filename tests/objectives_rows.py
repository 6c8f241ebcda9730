"""The gradients of the objectives on logits, element by element: what each element is in 64 bits and how far a kernel that
computes its exponentials in 32 may be from it, in proportion to the element itself. With u = 2^-24, d = (z - top) / tau and a
row's V logits:

  an exponential: the difference's rounding u |d|, the product's with log2 e u |d|, log2 e in 32 bits 0.3 u |d| (bf16 gradients
  leave out its low part), the exponential's ulp and the products behind it, 12 u in all
  their sum, in 64 bits: the mean of that over the softmax, where the mean of |d| is at most log V; a row that is walked scales
  what it has by the exponential of each new maximum's distance, a dozen times at most: 18 u more
  so log p of the target is off by the sum's error alone, and the ratios and coefficients by what that makes of them
"""

import math

import torch

U = 2.0 ** -24
TINY = 1e-37  # (32 bits have no more below it)


def _softmax(z, tau=1.0):
    """p, log p and each |d| of rows, p's relative error and the sum's; z - top first, so that no common size cancels."""
    z = z.double()
    d = (z - z.amax(-1, keepdim=True)) / tau
    log_s = torch.log(torch.exp(d).sum(-1, keepdim=True))
    logp = d - log_s
    far = torch.where(d > -1e4, d.abs(), 0.0)  # (further ones have p = 0 in any precision)
    own = U * (2.3 * far + 12)
    total = U * (2.3 * math.log(z.shape[-1]) + 30)
    return logp, own, total


def _pick(rows, y):
    return rows.gather(2, y[..., None])[..., 0]


def _onehot_grad(logp, own, total, y, on, c, dc, dtype):
    """c (onehot(y) - p) with c off by dc, and the tolerance."""
    c, dc = torch.where(on, c, 0.0)[..., None], torch.where(on, dc, 0.0)[..., None]
    p = logp.exp()
    rest = p.scatter(2, y[..., None], 0.0)
    one = rest.sum(-1, keepdim=True)                       # 1 - p of the target, without cancellation
    want = (-c * p).scatter(2, y[..., None], c * one)
    off = c.abs() * p * (own + total + 6 * U) + dc * p
    at = c.abs() * ((rest * own).sum(-1, keepdim=True) + one * (total + 6 * U) + 2.0 ** -50) + dc * one
    off = off.scatter(2, y[..., None], at)
    return want, off + torch.finfo(dtype).eps / 2 * want.abs() + TINY


def policy(logits, targets, mask, old_lp, adv, ref_lp=None, eps_lo=0.2, eps_hi=0.2, kl_coef=0.0, per="sequence", inv_n=None):
    """(dlogits, tolerance, the tokens where that holds: not those so close to a border of the clip that lp's error decides)."""
    B, T, V = logits.shape
    on = mask.bool() & (targets >= 0) & (targets < V)
    y = targets.clamp(0, V - 1)
    logp, own, total = _softmax(torch.where(on[..., None], logits, 0.0))
    lp = _pick(logp, y)
    r = torch.exp(lp - torch.where(on, old_lp.double(), 0.0))
    a = adv.double()[:, None] if adv.dim() == 1 else adv.double()
    a = torch.where(on, a.expand_as(lp), 0.0)
    lo, hi = 1 - eps_lo, 1 + eps_hi
    slope = torch.where(((a > 0) & (r > hi)) | ((a < 0) & (r < lo)), 0.0, a)
    sound = torch.minimum((r - lo).abs(), (r - hi).abs()) > 2 * r * total
    g, dg = -slope * r, (slope * r).abs() * (total + 6 * U)
    if ref_lp is not None:
        x = torch.where(on, ref_lp.double(), 0.0) - lp
        g = g - kl_coef * torch.expm1(x)
        dg = dg + abs(kl_coef) * (x.exp() * total + 6 * U * torch.expm1(x).abs())
    n = on.double()
    if per == "sequence":
        w = (1.0 / max(B, 1) if inv_n is None else inv_n) * n / n.sum(1, keepdim=True).clamp(min=1)
    else:
        w = n / n.sum().clamp(min=1) if inv_n is None else inv_n * n
    return (*_onehot_grad(logp, own, total, y, on, w * g, w * dg, logits.dtype), sound | ~on)


def preference(logits, targets, mask, ref_lp=None, pairs=None, beta=0.1, target=0.0, smoothing=0.0, lengths=None, inv_n=None):
    """(dlogits, tolerance, margin, tolerance)."""
    B, T, V = logits.shape
    on = mask.bool() & (targets >= 0) & (targets < V)
    y = targets.clamp(0, V - 1)
    logp, own, total = _softmax(torch.where(on[..., None], logits, 0.0))
    ratio = torch.where(on, _pick(logp, y) - (0.0 if ref_lp is None else ref_lp.double()), 0.0)
    size = torch.ones(B, dtype=torch.float64, device=logits.device) if lengths is None else lengths.double()
    s, ds = ratio.sum(1) / size, on.sum(1) * total / size
    if pairs is None:
        pairs = torch.arange(B, device=logits.device).view(-1, 2)
    P = pairs.shape[0]
    good = ((pairs >= 0) & (pairs < B)).all(1)
    c, r = pairs.clamp(0, B - 1).unbind(1)
    h = torch.where(good, beta * (s[c] - s[r]) - target, 0.0)
    dh = beta * (ds[c] + ds[r])
    step = beta * (1.0 / max(P, 1) if inv_n is None else inv_n)
    slope = torch.where(good, step * (smoothing * torch.sigmoid(h) - (1 - smoothing) * torch.sigmoid(-h)), 0.0)
    off = torch.where(good, step * dh / 4, 0.0)  # (the logistic function's slope is 1 / 4 at most)
    coef, dcoef = torch.zeros_like(s), torch.zeros_like(s)
    coef.index_add_(0, c, slope).index_add_(0, r, -slope)
    dcoef.index_add_(0, c, off).index_add_(0, r, off)
    coef, dcoef = (coef / size)[:, None].expand(B, T), (dcoef / size)[:, None].expand(B, T)
    dcoef = dcoef + 4 * U * coef.abs()
    return (*_onehot_grad(logp, own, total, y, on, coef, dcoef, logits.dtype), h, dh + 2 * U * h.abs())


def distill(logits, values, ids, t_lse=None, weights=None, temperature=1.0, inv_n=None):
    """(dlogits, tolerance, kl, tolerance)."""
    B, T, V = logits.shape
    tau = temperature
    w = torch.ones(B, T, dtype=torch.float64, device=logits.device) if weights is None else weights.double()
    on = w > 0
    logp, own, total = _softmax(torch.where(on[..., None], logits, 0.0), tau)
    there = on[..., None] & (ids >= 0) & (ids < V) & (values > -math.inf)
    at = ids.long().clamp(0, V - 1)
    t = torch.where(there, values.double(), -math.inf)
    if t_lse is None:
        d = (t - t.amax(-1, keepdim=True).clamp(min=-3.5e38)) / tau
        log_q = d - torch.log(torch.exp(d).sum(-1, keepdim=True))
        qrel = U * (2.3 * torch.where(d > -1e4, d.abs(), 0.0) + 12)
    else:
        log_q = t / tau - torch.where(on, t_lse.double(), 0.0)[..., None]
        qrel = torch.full_like(t, 8 * U)
    q = torch.where(there, torch.exp(log_q), 0.0)
    some = q > 0
    if t_lse is None:
        qrel = qrel + (q * qrel).sum(-1, keepdim=True) + 4 * U
    mass, dmass = q.sum(-1, keepdim=True), (q * qrel).sum(-1, keepdim=True)
    gap = torch.where(some, log_q - logp.gather(2, at), 0.0)
    kl = (q * gap).sum(-1)
    dkl = (q * qrel * gap.abs()).sum(-1) + (mass * total + dmass)[..., 0] + 2 * U * kl.abs() + TINY
    w = torch.where(on, w, 0.0)
    c = (w / w.sum() if inv_n is None and bool(w.sum() > 0) else w * (inv_n or 0.0))[..., None] * tau
    p = logp.exp()
    want = c * mass * p
    off = want * (own + total + 8 * U) + c * dmass * p
    want = want.scatter_add(2, at, -c * q)
    off = off.scatter_add(2, at, c * q * (qrel + 4 * U))
    empty = mass == 0
    want, off = torch.where(empty, 0.0, want), torch.where(empty, 0.0, off)
    return want, off + torch.finfo(logits.dtype).eps / 2 * want.abs() + TINY, torch.where(empty[..., 0], 0.0, kl), dkl


def outside(got, want, tol):
    """Which elements are too far (NaN is where none is wanted)."""
    return ~((got.double() - want).abs() <= tol)
