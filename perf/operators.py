"""The vocabulary's two ends at the k-mer vocabularies past 4-mers (k = 5 .. 8: 1367, 5463, 21847, 87383 tokens), as
cases to be timed and compared: the token embedding with its gradient, and the rules on logits with the token choice.

Kinds of case, each one call of one operator:
  lookup    embed_lookup: scaled embedding rows of n tokens
  gradient  embed_grad_sorted: the table's gradient from the rows' gradients, n rows of d
  process   process_logits: penalties for repeated tokens, bias and grammar mask on the logits of B sequences
  choose    choose_tokens: the same rules, then the token choice and its log-probability; nothing else written

With `own` false `run` computes them in elementary torch operations, in 32 bits (sums of gradients, log-probabilities and
Gumbel scores in 64); with `own` true it calls the framework.
"""

import math

import torch

own = False

DEV = "cuda"
N_SPECIAL, PAD, BOS, EOS = 3, 0, 1, 2
VOCABS = (1367, 5463, 21847, 87383)
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
MOST_ROWS = 512 * 1024   # a rollout's tokens: 512 sequences x 1024
MOST_BATCH = 512


def listed():
    return [
        # the embedding of one decode step: the last token of 64 sequences, 8-mers; a launch's latency
        {"name": "lookup_step", "kind": "lookup", "n": 64, "V": 87383, "d": 512, "weight": "bf16", "out": "bf16",
         "scale": 1.0},
        # a ragged micro-batch's token rows out of a bf16 table, at a width that is no power of two
        {"name": "lookup_ragged", "kind": "lookup", "n": 40961, "V": 21847, "d": 1000, "weight": "bf16", "out": "bf16",
         "scale": 31.622776},
        # a whole rollout's tokens (512 sequences x 1024) from the fp32 master table, 6-mers
        {"name": "lookup_rollout", "kind": "lookup", "n": 524288, "V": 5463, "d": 512, "weight": "fp32", "out": "fp32",
         "scale": 22.627417},
        # a few short calls of 5-mers: the gradient of an interactive fine-tuning step
        {"name": "gradient_short", "kind": "gradient", "n": 1003, "V": 1367, "d": 512, "rows": "fp32", "pad": True,
         "scale": 1.0},
        # a micro-batch of 32 calls, 7-mers, bf16 row gradients at a larger width
        {"name": "gradient_micro", "kind": "gradient", "n": 98305, "V": 21847, "d": 768, "rows": "bf16", "pad": False,
         "scale": 27.712813},
        # a rollout's tokens, 8-mers, the fp32 residual's gradient
        {"name": "gradient_rollout", "kind": "gradient", "n": 524288, "V": 87383, "d": 512, "rows": "fp32",
         "pad": True, "scale": 1.0},
        # one sequence's step with the 6-mer vocabulary: latency
        {"name": "process_single", "kind": "process", "B": 1, "V": 5463, "T": 300, "logits": "fp32", "out": "fp32"},
        # a served batch, 8-mers, bf16 logits in and out
        {"name": "process_batch", "kind": "process", "B": 512, "V": 87383, "T": 256, "logits": "bf16", "out": "bf16"},
        # one sequence's greedy step, 8-mers: the vocabulary spread over the chip, then joined
        {"name": "choose_single", "kind": "choose", "B": 1, "V": 87383, "T": 1024, "logits": "fp32", "mode": "greedy"},
        # a ragged batch's sampled step, 7-mers: Gumbel noise from one uniform per vocabulary entry
        {"name": "choose_sampled", "kind": "choose", "B": 77, "V": 21847, "T": 411, "logits": "bf16", "mode": "gumbel"},
        # the rollout's batch, greedy, 8-mers, fp32 logits as the head writes them
        {"name": "choose_rollout", "kind": "choose", "B": 512, "V": 87383, "T": 256, "logits": "fp32", "mode": "greedy"},
        # the rollout's batch, sampled, 6-mers
        {"name": "choose_kmer6", "kind": "choose", "B": 512, "V": 5463, "T": 341, "logits": "fp32", "mode": "gumbel"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """Vocabularies of 343 to 87383 tokens; 1 to 524288 rows of 64 to 1024 columns (odd widths among them); batches of 1
    to 512 sequences with histories of 1 to 2048 tokens."""
    kind = rng.choice(["lookup", "gradient", "process", "choose"])
    V = rng.choice(VOCABS) if rng.random() < 0.5 else _log_uniform(rng, 343, VOCABS[-1])
    if kind in ("lookup", "gradient"):
        d = 64 * rng.randint(1, 16) if rng.random() < 0.6 else _log_uniform(rng, 64, 1024)
        n = min(_log_uniform(rng, 1, MOST_ROWS), (MOST_ROWS * 512) // d)
        case = {"kind": kind, "n": n, "V": V, "d": d, "scale": rng.choice([1.0, math.sqrt(d), 0.125])}
        if kind == "lookup":
            w = rng.choice(["bf16", "fp32"])
            return {**case, "weight": w, "out": rng.choice([w, "bf16", "fp32"])}
        return {**case, "rows": rng.choice(["bf16", "fp32"]), "pad": rng.random() < 0.5}
    case = {"kind": kind, "B": _log_uniform(rng, 1, MOST_BATCH), "V": V, "T": _log_uniform(rng, 1, 2048),
            "logits": rng.choice(["bf16", "fp32"])}
    if kind == "process":
        return {**case, "out": rng.choice([case["logits"], "fp32"])}
    return {**case, "mode": rng.choice(["greedy", "gumbel"])}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _tokens(shape, V, g):
    """Token ids as reads have them: k-mers of an uneven base composition (some hundreds of times as frequent as others)."""
    u = torch.rand(shape, generator=g, device=DEV)
    return N_SPECIAL + (u.pow(2.5) * (V - N_SPECIAL)).long().clamp_(max=V - N_SPECIAL - 1)


def _rules(B, V, T, g):
    """Histories and rules of a batch of requests: each sequence its own length (0 among them), penalties and grammar
    state. Grammar rows: everything but PAD and BOS; only EOS (after a tail token); a random half; nothing but PAD."""
    hist = _tokens((B, T), V, g)
    again = torch.randint(0, T, (B, T), generator=g, device=DEV)  # repeats, as low-complexity reads have them
    hist = torch.where(torch.rand(B, T, generator=g, device=DEV) < 0.3, hist.gather(1, again), hist)
    lengths = torch.randint(0, T + 1, (B,), generator=g, device=DEV).int()
    pick = torch.rand(B, generator=g, device=DEV)
    rep = torch.where(pick < 0.3, torch.ones_like(pick), 1.0 + 0.4 * torch.rand(B, generator=g, device=DEV))
    pres = 0.7 * torch.rand(B, generator=g, device=DEV)
    freq = 0.3 * torch.rand(B, generator=g, device=DEV)
    bias = 0.5 * torch.randn(V, generator=g, device=DEV)
    bias[[PAD, BOS]] = float("-inf")
    allowed = torch.ones(4, V, dtype=torch.bool, device=DEV)
    allowed[0, [PAD, BOS]] = False
    allowed[1] = False
    allowed[1, EOS] = True
    allowed[2] = torch.rand(V, generator=g, device=DEV) < 0.5
    allowed[2, EOS] = True
    allowed[3] = False
    allowed[3, PAD] = True
    # -1: no mask for this sequence; the dead ends (EOS only, PAD only) are rare
    state = torch.tensor([-1, 0, 0, 0, 2, 2, 2, 1, 3], device=DEV)[torch.randint(0, 9, (B,), generator=g, device=DEV)]
    bits = torch.zeros(4, -(-V // 32) * 32, dtype=torch.int64, device=DEV)
    bits[:, :V] = allowed
    words = (bits.view(4, -1, 32) << torch.arange(32, device=DEV)).sum(-1)
    packed = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()  # bit v % 32 of word v // 32
    return {"history": hist, "lengths": lengths, "repetition": rep, "presence": pres, "frequency": freq, "bias": bias,
            "allowed": packed, "allowed_rows": state.int()}


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    kind, V = case["kind"], case["V"]
    if kind == "lookup":
        w = torch.randn(V, case["d"], generator=g, device=DEV).mul_(0.02).to(TYPES[case["weight"]])
        return {"case": case, "weight": w, "tokens": _tokens((case["n"],), V, g)}
    if kind == "gradient":
        n = case["n"]
        tok = _tokens((n,), V, g)
        # calls end at different lengths: the last fifth of each row of 128 is padding
        tok = torch.where(torch.arange(n, device=DEV) % 128 >= 102, torch.full_like(tok, PAD), tok)
        rows = torch.randn(n, case["d"], generator=g, device=DEV).to(TYPES[case["rows"]])
        return {"case": case, "rows": rows, "tokens": tok}
    B = case["B"]
    z = torch.randn(B, V, generator=g, device=DEV).mul_(3).to(TYPES[case["logits"]])
    state = {"case": case, "logits": z, "rules": _rules(B, V, case["T"], g)}
    if kind == "choose":
        sampled = case["mode"] == "gumbel"
        state["temperature"] = (0.6 + 0.7 * torch.rand(B, generator=g, device=DEV)) if sampled else 0.0
        state["uniforms"] = torch.rand(B, V, generator=g, device=DEV) if sampled else None
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------

def _plain_rules(x, r):
    """fp32 logits after the rules: repetition, frequency, presence, bias, mask; each step rounded to 32 bits."""
    B, V = x.shape
    z = x.float()
    hist, T = r["history"], r["history"].shape[1]
    live = torch.arange(T, device=DEV)[None, :] < r["lengths"][:, None]
    count = torch.zeros(B, V, dtype=torch.int32, device=DEV).scatter_add_(1, hist, live.int())
    seen = count > 0
    rep = r["repetition"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - r["frequency"][:, None] * count.float()
    z = z - torch.where(seen, r["presence"][:, None], 0.0)
    z = z + r["bias"]
    word = torch.arange(V, device=DEV)
    row = r["allowed_rows"].long()
    bit = (r["allowed"][row.clamp(min=0)][:, word // 32] >> (word % 32).int()) & 1
    return torch.where((bit == 1) | (row < 0)[:, None], z, float("-inf"))


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "lookup":
        return (s["weight"][s["tokens"]].float() * case["scale"]).to(TYPES[case["out"]])
    if kind == "gradient":
        # in token order, each token's rows summed as a difference of running sums (64 bits: the sums get long)
        tok, order = torch.sort(s["tokens"], stable=True)
        upto = s["rows"][order].t().double().cumsum(1)
        ends = torch.searchsorted(tok, torch.arange(case["V"], device=DEV), right=True)
        upto = torch.where(ends > 0, upto[:, (ends - 1).clamp(min=0)], 0.0)
        table = torch.diff(upto, dim=1, prepend=upto.new_zeros(case["d"], 1)) * case["scale"]
        if case["pad"]:
            table[:, PAD] = 0
        return table.t().float().contiguous()
    z = _plain_rules(s["logits"], s["rules"])
    if kind == "process":
        return z.to(TYPES[case["out"]])
    V = case["V"]
    if case["mode"] == "gumbel":
        z = z / s["temperature"][:, None]
        score = z.double() - torch.log(-torch.log(s["uniforms"].double().clamp(min=1e-20)))
    else:
        score = z
    best = score.max(1, keepdim=True).values
    tok = torch.where(score == best, torch.arange(V, device=DEV), V).min(1).values  # ties: the lowest id
    tok = torch.where(best[:, 0] == float("-inf"), torch.zeros_like(tok), tok)      # nothing allowed: the fallback, 0
    top = z.max(1, keepdim=True).values.clamp(min=-3e38)
    lse = torch.log(torch.exp(z.double() - top.double()).sum(1)) + top[:, 0].double()
    logp = z.gather(1, tok[:, None])[:, 0].double() - lse
    return tok, torch.where(best[:, 0] == float("-inf"), torch.full_like(logp, float("-inf")), logp).float()


def run(state):
    if not own:
        return _plain(state)
    from viktor_amd import hip_ops as ops
    case = state["case"]
    kind = case["kind"]
    if kind == "lookup":
        return ops.embed_lookup(state["weight"], state["tokens"], scale=case["scale"], out_dtype=TYPES[case["out"]])
    if kind == "gradient":
        return ops.embed_grad_sorted(state["rows"], state["tokens"], case["V"], scale=case["scale"],
                                     pad=PAD if case["pad"] else None)
    if kind == "process":
        return ops.process_logits(state["logits"], out_dtype=TYPES[case["out"]], **state["rules"])
    return ops.choose_tokens(state["logits"], temperature=state["temperature"], uniforms=state["uniforms"],
                             **state["rules"])


def work(case):
    kind, V = case["kind"], case["V"]
    if kind == "lookup":
        n, d = case["n"], case["d"]
        # the rows that n ids can touch, once each
        return {"bytes": n * 8 + min(n, V) * d * SIZE[case["weight"]] + n * d * SIZE[case["out"]], "flops": n * d}
    if kind == "gradient":
        n, d = case["n"], case["d"]
        used = n * 102 // 128 if case["pad"] else n  # padding rows are not read
        return {"bytes": n * 8 + used * d * SIZE[case["rows"]] + V * d * 4, "flops": used * d}
    B, T = case["B"], case["T"]
    rules = B * T * 4 + V * 4 + 4 * V // 8  # half of each history is in use, 8 bytes a token
    if kind == "process":
        return {"bytes": B * V * (SIZE[case["logits"]] + SIZE[case["out"]]) + rules, "flops": 6 * B * V}
    noise = 4 * B * V if case["mode"] == "gumbel" else 0
    return {"bytes": B * V * SIZE[case["logits"]] + noise + rules + 12 * B, "flops": 12 * B * V}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind, V = case["kind"], case["V"]
    if kind == "lookup":
        d = case["d"]
        flat = s["weight"].double().reshape(-1)
        at = s["tokens"][:, None] * d + torch.arange(d, device=DEV)
        return torch.take(flat, at) * case["scale"]
    if kind == "gradient":
        rows = s["rows"].double()
        if case["pad"]:
            rows[s["tokens"] == PAD] = 0
        return torch.zeros(V, case["d"], dtype=torch.float64, device=DEV).index_add_(0, s["tokens"], rows) * case["scale"]
    r = s["rules"]
    out, toks, lps = [], [], []
    for b in range(case["B"]):
        z = s["logits"][b].double()
        past = r["history"][b, :int(r["lengths"][b])]
        ids, times = torch.unique(past, return_counts=True)
        old = z[ids]
        rep = r["repetition"][b].double()
        new = torch.where(old > 0, old / rep, old * rep)
        z[ids] = new - r["frequency"][b].double() * times - r["presence"][b].double()
        z = z + r["bias"].double()
        row = int(r["allowed_rows"][b])
        if row >= 0:
            v = torch.arange(V, device=DEV)
            words = r["allowed"][row].long() & 0xffffffff
            z[((words[v >> 5] >> (v & 31)) & 1) == 0] = -math.inf
        if kind == "process":
            out.append(z)
            continue
        noise = 0.0
        if case["mode"] == "gumbel":
            z = z / s["temperature"][b].double()
            noise = -torch.log(-torch.log(s["uniforms"][b].double().clamp(min=1e-20)))
        tok = torch.argmax(z + noise) if bool((z > -math.inf).any()) else torch.zeros((), dtype=torch.long, device=DEV)
        toks.append(tok)
        lps.append(torch.log_softmax(z, 0)[tok] if bool((z > -math.inf).any()) else z.new_tensor(-math.inf))
    return torch.stack(out) if kind == "process" else (torch.stack(toks), torch.stack(lps))
