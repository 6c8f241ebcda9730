"""Objectives on the decoder's logits, as cases to be timed and compared: what a policy update, a preference update and a
distillation do between the LM head's product and its backward, at the vocabularies from single bases (7) to 8-mers (87383).

Kinds of case, each one call of one operator on the logits [B, T, V] of B teacher-forced calls:
  policy      policy_score / token_policy_loss: clipped policy loss per token with a KL term, and its gradient
  preference  preference_score / preference_loss: the loss of paired log ratios, and its gradient
  top         top_logits: each token's k largest logits with their ids, and the log-sum-exp (a teacher's list)
  distill     distill_score / distill_loss: divergence from a teacher's list, and its gradient

"call" says by which entry point: "score" returns the gradient beside the loss, "loss" is differentiable and followed by
its backward pass. With `own` false `run` computes the same in elementary torch operations, in 32 bits (sums, log-ratios
and what is next to the clip's borders in 64); with `own` true it calls the framework.
"""

import math

import torch

own = False

DEV = "cuda"
N_SPECIAL, PAD = 3, 0
VOCABS = (7, 343, 1367, 5463, 21847, 87383)
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
MOST_LOGITS = 2064 * 87383
MOST_TOKENS = 512 * 1024   # a rollout's: 512 sequences x 1024
MOST_LIST = 128
EPS_LO, EPS_HI, KL_COEF, BETA = 0.2, 0.28, 0.04, 0.1


def listed():
    return [
        # a few short calls of 5-mers: an interactive fine-tuning step, launches and host calls
        {"name": "policy_short", "kind": "policy", "call": "score", "B": 4, "T": 37, "V": 1367, "logits": "fp32",
         "ref": True, "per": "sequence"},
        # the rollout of single bases: 512 calls of 1024 tokens
        {"name": "policy_bases", "kind": "policy", "call": "score", "B": 512, "T": 1024, "V": 7, "logits": "bf16",
         "ref": True, "per": "token"},
        # a ragged micro-batch of 6-mers (1024 bases in 171 tokens), as an update runs it: loss, then backward
        {"name": "policy_kmer6", "kind": "policy", "call": "loss", "B": 96, "T": 171, "V": 5463, "logits": "bf16",
         "ref": True, "per": "sequence"},
        # two pairs of short 4-mer calls
        {"name": "preference_short", "kind": "preference", "call": "score", "B": 4, "T": 65, "V": 343, "logits": "fp32",
         "pairs": 0, "smooth": 0.0},
        # 64 windows with a better and a worse call each, 4-mers
        {"name": "preference_kmer4", "kind": "preference", "call": "loss", "B": 128, "T": 257, "V": 343, "logits": "bf16",
         "pairs": 0, "smooth": 0.1},
        # groups of calls with several pairs among them, 7-mers: sequences in more than one pair
        {"name": "preference_kmer7", "kind": "preference", "call": "score", "B": 32, "T": 147, "V": 21847,
         "logits": "bf16", "pairs": 48, "smooth": 0.0},
        # a served teacher: the lists of 8 tokens of one decode batch
        {"name": "top_step", "kind": "top", "B": 8, "T": 1, "V": 5463, "logits": "fp32", "k": 16, "tau": 1.0},
        # a teacher's lists of a micro-batch, 4-mers
        {"name": "top_kmer4", "kind": "top", "B": 128, "T": 257, "V": 343, "logits": "bf16", "k": 32, "tau": 1.0},
        # a teacher's lists of a micro-batch, 8-mers
        {"name": "top_kmer8", "kind": "top", "B": 16, "T": 129, "V": 87383, "logits": "bf16", "k": 64, "tau": 2.0},
        # three short calls of 4-mers against lists of 8
        {"name": "distill_short", "kind": "distill", "call": "score", "B": 3, "T": 50, "V": 343, "logits": "bf16", "k": 8,
         "list": "fp32", "tau": 1.0, "lse": False},
        # a micro-batch of 6-mers, the teacher's own probabilities (its log-sum-exp kept)
        {"name": "distill_kmer6", "kind": "distill", "call": "loss", "B": 96, "T": 171, "V": 5463, "logits": "bf16",
         "k": 64, "list": "bf16", "tau": 1.0, "lse": True},
        # a micro-batch of 8-mers with fp32 logits, softened, lists renormalised
        {"name": "distill_kmer8", "kind": "distill", "call": "score", "B": 16, "T": 129, "V": 87383, "logits": "fp32",
         "k": 32, "list": "fp32", "tau": 2.0, "lse": False},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """Vocabularies of 7 to 87383 tokens (odd ones among them), 1 to 512 sequences of 1 to 1024 tokens, lists of 1 to 128."""
    kind = rng.choice(["policy", "preference", "top", "distill"])
    V = rng.choice(VOCABS) if rng.random() < 0.5 else _log_uniform(rng, 7, VOCABS[-1])
    most = max(2, min(MOST_TOKENS, MOST_LOGITS // V))
    n = _log_uniform(rng, 2, most)
    B = _log_uniform(rng, 2 if kind == "preference" else 1, max(2, min(512, n)))
    B -= B % 2 if kind == "preference" else 0
    T = max(1, min(1024, n // B))
    case = {"kind": kind, "B": B, "T": T, "V": V, "logits": rng.choice(["bf16", "fp32"])}
    if kind != "top":
        case["call"] = rng.choice(["score", "loss"])
    if kind == "policy":
        return {**case, "ref": rng.random() < 0.7, "per": rng.choice(["sequence", "token"])}
    if kind == "preference":
        return {**case, "pairs": rng.choice([0, _log_uniform(rng, 1, 4 * B)]), "smooth": rng.choice([0.0, 0.1])}
    case["k"] = _log_uniform(rng, 1, min(MOST_LIST, V))
    case["tau"] = rng.choice([1.0, 1.0, 2.0, 0.7])
    if kind == "top":
        return case
    return {**case, "list": rng.choice(["bf16", "fp32"]), "lse": rng.random() < 0.5}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _calls(case, g):
    """Logits of B teacher-forced calls with their targets and the mask of their tokens: calls end at different lengths
    (half of T to all of it), PAD behind. The model is fairly sure of most targets, as a trained one is."""
    B, T, V = case["B"], case["T"], case["V"]
    u = torch.rand(B, T, generator=g, device=DEV)
    y = N_SPECIAL + (u.pow(2.5) * (V - N_SPECIAL)).long().clamp_(max=V - N_SPECIAL - 1)
    ends = torch.randint((T + 1) // 2, T + 1, (B, 1), generator=g, device=DEV)
    mask = torch.arange(T, device=DEV) < ends
    z = torch.randn(B, T, V, generator=g, device=DEV).mul_(2)
    sure = math.log(V) + 2 + 3 * torch.rand(B, T, 1, generator=g, device=DEV)
    sure = torch.where(torch.rand(B, T, 1, generator=g, device=DEV) < 0.1, 0.0, sure)
    z.scatter_add_(2, y[..., None], sure)
    z = z.to(TYPES[case["logits"]])
    return z, torch.where(mask, y, PAD), mask


def _drifted(lp, g, mean=0.0):
    """Log-probabilities of a policy some steps away: most within a few percent, some far."""
    far = torch.rand(lp.shape, generator=g, device=DEV) < 0.02
    drift = torch.randn(lp.shape, generator=g, device=DEV) * torch.where(far, 0.4, 0.03)
    return (lp + drift + mean).clamp(max=0.0)


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    kind, B, T, V = case["kind"], case["B"], case["T"], case["V"]
    z, y, mask = _calls(case, g)
    s = {"case": case, "logits": z}
    if kind in ("policy", "preference"):
        lse = torch.cat([torch.logsumexp(part.float(), -1) for part in z.split(max(1, (1 << 26) // (T * V)))])
        lp = (z.gather(2, y[..., None])[..., 0].float() - lse) * mask
        s |= {"targets": y, "mask": mask}
    if kind == "policy":
        s["old_lp"] = _drifted(lp, g) * mask
        s["ref_lp"] = _drifted(lp, g) * mask if case["ref"] else None
        s["adv"] = torch.randn(B, generator=g, device=DEV)
    elif kind == "preference":
        # the update has moved each call's tokens by a mean of its own
        s["ref_lp"] = _drifted(lp, g, 4.0 / T * torch.randn(B, 1, generator=g, device=DEV)) * mask
        if case["pairs"]:
            first = torch.randint(0, B, (case["pairs"],), generator=g, device=DEV)
            other = (first + torch.randint(1, B, (case["pairs"],), generator=g, device=DEV)) % B
            s["pairs"] = torch.stack([first, other], 1)
        else:
            s["pairs"] = None
    elif kind == "distill":
        t = z.float() + 0.7 * torch.randn(B, T, V, generator=g, device=DEV)
        val, ids = torch.topk(t, case["k"], -1)
        s["t_lse"] = torch.logsumexp(t / case["tau"], -1) if case["lse"] else None
        del t
        # some lists are shorter: id -1 behind their end
        short = torch.randint(1, case["k"] + 1, (B, T, 1), generator=g, device=DEV)
        short = torch.where(torch.rand(B, T, 1, generator=g, device=DEV) < 0.25, short, case["k"])
        s["t_ids"] = torch.where(torch.arange(case["k"], device=DEV) < short, ids, -1).int()
        s["t_values"] = val.to(TYPES[case["list"]])
        s["weights"] = torch.where(mask, 0.25 + torch.rand(B, T, generator=g, device=DEV), 0.0)
    if case.get("call") == "loss":
        s["logits"].requires_grad_(True)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------

def _softmax_parts(z):
    """exp(z - max), the maxima and the sums (64 bits) of rows."""
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    return e, top, e.sum(-1, keepdim=True, dtype=torch.float64)


def _gradient(e, total, y, coef, dtype):
    """coef (onehot(y) - softmax) of rows with exponentials e."""
    d = e * (-coef / total).float()
    d.scatter_add_(2, y[..., None], coef.float())
    return d.to(dtype)


def _plain_policy(s):
    case, y, on = s["case"], s["targets"], s["mask"]
    logits = s["logits"].detach()
    z = logits.float()
    e, top, total = _softmax_parts(z)
    lp = ((z.gather(2, y[..., None]) - top).double() - torch.log(total))[..., 0]
    a = s["adv"].double()[:, None]
    r = torch.exp(lp - s["old_lp"].double())
    inside = (r >= 1 - EPS_LO) & (r <= 1 + EPS_HI)
    free, cut = r * a, r.clamp(1 - EPS_LO, 1 + EPS_HI) * a
    pg = -torch.minimum(free, cut)
    slope = torch.where(free < cut, a, torch.where(cut < free, a * inside, (a + a * inside) / 2))
    g = -r * slope
    kl = None
    loss = pg
    if s["ref_lp"] is not None:
        x = s["ref_lp"].double() - lp
        kl = torch.expm1(x) - x
        loss = loss + KL_COEF * kl
        g = g - KL_COEF * torch.expm1(x)
        kl = torch.where(on, kl, 0.0).float()
    if case["per"] == "sequence":
        w = 1.0 / case["B"] / on.sum(1, keepdim=True).clamp(min=1).double()
    else:
        w = 1.0 / on.sum().clamp(min=1).double()
    coef = torch.where(on, w * g, 0.0)[..., None]
    loss = torch.where(on, w * loss, 0.0).sum().float()
    d = _gradient(e, total, y, coef, logits.dtype)
    return loss, torch.where(on, pg, 0.0).float(), kl, torch.where(on, lp, 0.0).float(), d


def _plain_preference(s):
    case, y, on = s["case"], s["targets"], s["mask"]
    logits = s["logits"].detach()
    z = logits.float()
    e, top, total = _softmax_parts(z)
    lp = ((z.gather(2, y[..., None]) - top).double() - torch.log(total))[..., 0]
    ratio = torch.where(on, lp - s["ref_lp"].double(), 0.0).sum(1)
    pairs = s["pairs"]
    if pairs is None:
        pairs = torch.arange(case["B"], device=DEV).view(-1, 2)
    n, eps = pairs.shape[0], case["smooth"]
    h = BETA * (ratio[pairs[:, 0]] - ratio[pairs[:, 1]])
    soft = lambda x: x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))  # noqa: E731
    loss = ((1 - eps) * soft(-h) + eps * soft(h)).sum() / n
    dh = BETA / n * (1 / (1 + torch.exp(-h)) - (1 - eps))
    c = torch.zeros_like(ratio).index_add_(0, pairs[:, 0], dh).index_add_(0, pairs[:, 1], -dh)
    coef = torch.where(on, c[:, None], 0.0)[..., None]
    return loss.float(), h.float(), torch.where(on, lp, 0.0).float(), _gradient(e, total, y, coef, logits.dtype)


def _plain_top(s):
    case = s["case"]
    val, ids = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    z = s["logits"].float() / case["tau"]
    _, top, total = _softmax_parts(z)
    lse = (top.double() + torch.log(total))[..., 0].float()
    return val[..., :case["k"]].contiguous(), ids[..., :case["k"]].int(), lse


def _plain_distill(s):
    case, w, tau = s["case"], s["weights"].double(), s["case"]["tau"]
    logits = s["logits"].detach()
    z = logits.float() / tau
    e, top, total = _softmax_parts(z)
    there = s["t_ids"] >= 0
    at = s["t_ids"].long().clamp(min=0)
    t = torch.where(there, s["t_values"].double() / tau, float("-inf"))
    if s["t_lse"] is None:
        lead = t.amax(-1, keepdim=True)
        log_q = t - lead - torch.log(torch.exp(t - lead).sum(-1, keepdim=True))
        mass = torch.ones_like(lead)
    else:
        log_q = t - s["t_lse"].double()[..., None]
        mass = torch.exp(log_q).sum(-1, keepdim=True)
    q = torch.exp(log_q)
    log_p = (z.gather(2, at) - top).double() - torch.log(total)
    kl = torch.where(there, q * (log_q - log_p), 0.0).sum(-1)
    share = torch.where(w > 0, w / w.sum().clamp(min=1e-300), 0.0)[..., None] * tau
    d = e * (share * mass / total).float()
    d.scatter_add_(2, at, (-share * q).float())
    kl = torch.where(w > 0, kl, 0.0)
    return (tau * share[..., 0] * kl).sum().float(), kl.float(), d.to(logits.dtype)


def _plain(s):
    return {"policy": _plain_policy, "preference": _plain_preference, "top": _plain_top,
            "distill": _plain_distill}[s["case"]["kind"]](s)


def run(state):
    if not own:
        return _plain(state)
    from viktor_amd import hip_ops as ops, objectives
    s, case = state, state["case"]
    kind = case["kind"]
    if kind == "top":
        return ops.top_logits(s["logits"], case["k"], temperature=case["tau"])
    if kind == "policy":
        args = (s["logits"], s["targets"], s["mask"], s["old_lp"], s["adv"])
        more = {"ref_lp": s["ref_lp"], "eps_lo": EPS_LO, "eps_hi": EPS_HI, "kl_coef": KL_COEF if case["ref"] else 0.0,
                "per": case["per"]}
        if case["call"] == "score":
            r = ops.policy_score(*args, **more)
            return r["loss"], r["pg"], r["kl"], r["lp"], r["dlogits"]
        out = objectives.token_policy_loss(*args, **more)
    elif kind == "preference":
        args = (s["logits"], s["targets"], s["mask"], s["ref_lp"])
        more = {"pairs": s["pairs"], "beta": BETA, "smoothing": case["smooth"]}
        if case["call"] == "score":
            r = ops.preference_score(*args, **more)
            return r["loss"], r["margin"], r["lp"], r["dlogits"]
        out = objectives.preference_loss(*args, **more)
    else:
        args = (s["logits"], s["t_values"], s["t_ids"])
        more = {"t_lse": s["t_lse"], "weights": s["weights"], "temperature": case["tau"]}
        if case["call"] == "score":
            r = ops.distill_score(*args, **more)
            return r["loss"], r["kl"], r["dlogits"]
        out = objectives.distill_loss(*args, **more)
    return (*out, *torch.autograd.grad(out[0], s["logits"]))


def work(case):
    kind, V, L = case["kind"], case["V"], SIZE[case["logits"]]
    n = case["B"] * case["T"]
    if kind == "top":
        return {"bytes": n * (V * L + case["k"] * (L + 4) + 4), "flops": 4 * n * V}
    used = 3 * n // 4  # rows behind a call's end are not read; their gradients are zeros
    logits = (used + n) * V * L
    if kind == "distill":
        return {"bytes": logits + used * case["k"] * (SIZE[case["list"]] + 4) + n * 8 + 4 * n * case["lse"],
                "flops": 8 * used * V}
    per_token = 8 + 1 + 4 + 4 + (4 + 8 * case["ref"] if kind == "policy" else 0)
    return {"bytes": logits + n * per_token, "flops": 8 * used * V}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind, tau = case["kind"], case.get("tau", 1.0)
    if kind == "top":
        z = s["logits"].float()
        bits = z.view(torch.int32).long()
        order = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits)  # as the values compare (no zeros of either sign here)
        V = case["V"]
        key = (order << 20) + (V - 1 - torch.arange(V, device=DEV))    # equal values: the lower id first
        ids = V - 1 - (torch.topk(key, case["k"], -1).values & 0xfffff)
        return z.double().gather(2, ids), ids, torch.logsumexp(s["logits"].double() / tau, -1)
    z = s["logits"].detach().double().requires_grad_(True)
    logp = torch.log_softmax(z / tau, -1)
    if kind == "distill":
        t = (s["t_values"].double() / tau).masked_fill(s["t_ids"] < 0, -math.inf)
        log_q = torch.log_softmax(t, -1) if s["t_lse"] is None else t - s["t_lse"].double()[..., None]
        log_q = log_q.masked_fill(s["t_ids"] < 0, -1e4)  # a weight of exactly 0
        kl = (log_q.exp() * (log_q - logp.gather(2, s["t_ids"].long().clamp(min=0)))).sum(-1) * (s["weights"] > 0)
        w = s["weights"].double()
        loss = tau ** 2 * (w * kl).sum() / w.sum()
        return loss.detach(), kl.detach(), torch.autograd.grad(loss, z)[0]
    on = s["mask"].double()
    lp = logp.gather(2, s["targets"][..., None])[..., 0] * on
    if kind == "policy":
        r = torch.exp(lp - s["old_lp"].double())
        a = s["adv"].double()[:, None]
        pg = -torch.minimum(r * a, torch.clamp(r, 1 - EPS_LO, 1 + EPS_HI) * a)
        kl = None
        term = pg
        if case["ref"]:
            x = s["ref_lp"].double() - lp
            kl = torch.exp(x) - x - 1
            term = term + KL_COEF * kl
        if case["per"] == "sequence":
            loss = ((term * on).sum(1) / on.sum(1).clamp(min=1)).mean()
        else:
            loss = (term * on).sum() / on.sum().clamp(min=1)
        dz = torch.autograd.grad(loss, z)[0]
        return loss.detach(), (pg * on).detach(), None if kl is None else (kl * on).detach(), lp.detach(), dz
    ratio = (lp - s["ref_lp"].double() * on).sum(1)
    first, second = ratio[0::2], ratio[1::2]
    if s["pairs"] is not None:
        first, second = ratio[s["pairs"][:, 0]], ratio[s["pairs"][:, 1]]
    h = BETA * (first - second)
    log_s = torch.nn.functional.logsigmoid
    loss = -((1 - case["smooth"]) * log_s(h) + case["smooth"] * log_s(-h)).mean()
    return loss.detach(), h.detach(), lp.detach(), torch.autograd.grad(loss, z)[0]
