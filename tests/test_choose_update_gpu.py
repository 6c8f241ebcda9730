"""choose_update called directly, in every way a decode step can be cut: a whole row per workgroup, slices that a second
launch joins, the inverse CDF of slices, histories counted by token (more than 2048 output columns). Tokens and
log-probabilities against choose_tokens on the same rules (the same bits) and against the CPU's choice in fp64, the state
against a restatement of the step's rules (viktor/engine.py:79-116) on the host, over several steps and in a graph."""

import numpy as np
import pytest
import torch

from tests.test_engine_gpu import check_stream, run_case
from tests.test_vocab_gpu import _choice_ref, _rules_ref, _tame
from viktor_amd import hip_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
PAD, BOS, EOS = 0, 1, 2
STOP = 4                      # the homopolymer rule's run, in tokens
PENALTIES = (1.25, 0.5, 0.25)  # exact in fp32
STATE = ("tok", "run", "pos", "out", "logp", "pos32", "seqlens", "rpos32")


def _problem(B, V, T, dt, seed, gumbel):
    """A batch in the middle of decoding. Output columns: 0, one in the middle, the last, past it, then any. Rows that are
    over, behind a tail token, one short of the homopolymer rule, and without any allowed token, in turn."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    col = torch.randint(0, T, (B,), generator=g)
    col[:4] = torch.tensor([0, T // 2, T - 1, T + 2])[:B]
    plen = torch.randint(1, 50, (B,), generator=g)
    tail, homo = rnd(V) < 0.2, rnd(V) < 0.5
    tail[[PAD, BOS, EOS, 7, 9]] = homo[[PAD, BOS, EOS, 7, 9]] = False
    plain, behind, many = (20 + int(torch.nonzero(f[20:])[0]) for f in (~tail & ~homo, tail, homo & ~tail))
    tok = torch.tensor([plain, many, behind, EOS, 7, PAD, 9])[(torch.arange(B) + seed) % 7].contiguous()
    masks = rnd(4, V) < 0.5
    masks[2] = False            # nothing
    masks[:2, [plain, many]] = True
    masks[3] = True
    token_rows = torch.randint(-1, 2, (V,), generator=g).int()
    token_rows[7], token_rows[9], token_rows[many] = 2, 3, -1
    x = 3 * torch.randn(B, V, generator=g)
    x[torch.arange(B), tok] += torch.where(tok == many, 40.0, 0.0)  # (the run goes on, whatever the penalties)
    bias = torch.randn(V, generator=g)
    bias[[PAD, BOS]] = float("-inf")
    # what has been produced, and behind it other sequences' remains, which count nowhere
    hist = (rnd(B, T).pow(3) * (V - 3)).long() + 3
    s = {"tok": tok, "run": torch.where(tok == many, STOP - 2, 0).long(), "pos": plen + col, "plen": plen, "hist": hist,
         "rope": torch.randint(0, 9, (B,), generator=g), "base": torch.randint(0, 5, (B,), generator=g), "x": x.to(dt), "bias": bias,
         "tail": tail, "homo": homo, "masks": masks, "token_rows": token_rows}
    s["u"] = torch.rand(B, T, *((V,) if gumbel else ()), generator=torch.Generator(DEV).manual_seed(seed + 1), device=DEV)
    return s


def _device(s):
    """The call's tensors; out's rows are wider than its columns."""
    B, T = s["hist"].shape
    d = {k: s[k].to(DEV) for k in ("tok", "run", "pos", "plen", "rope", "base", "bias", "tail", "homo", "token_rows")}
    d["out"] = torch.full((B, T + 5), -3, dtype=torch.long, device=DEV)[:, :T]
    d["out"].copy_(s["hist"])
    d["logp"] = torch.full((B, T), 7.0, device=DEV)
    for k in ("pos32", "seqlens", "rpos32"):
        d[k] = torch.zeros(B, dtype=torch.int32, device=DEV)
    d["allowed"] = ops.pack_allowed(s["masks"]).to(DEV)
    return d


def _step(d, x, temperature, u, rules):
    kw = dict(zip(("repetition", "presence", "frequency"), PENALTIES)) if rules else {}
    ops.choose_update(x, d["bias"], d["tail"], d["homo"], STOP, d["tok"], d["run"], d["pos"], d["plen"], d["rope"], d["out"],
                      d["pos32"], d["seqlens"], d["rpos32"], EOS, PAD, temperature=temperature, uniforms=u,
                      gumbel=u is not None and u.dim() == 3, logp_out=d["logp"], cache_base=d["base"], allowed=d["allowed"] if rules else None,
                      token_rows=d["token_rows"] if rules else None, **kw)


def _advance(h, s, chosen, logp, T):
    """One step's rules on the host: what is forced, written and counted."""
    for b in range(len(chosen)):
        prev, nxt, col = int(h["tok"][b]), int(chosen[b]), int(h["pos"][b] - s["plen"][b])
        if 0 <= col < T:
            h["logp"][b, col] = logp[b]
        if s["tail"][prev]:
            nxt = EOS
        h["run"][b] = h["run"][b] + 1 if nxt == prev and s["homo"][nxt] else 0
        if h["run"][b] + 1 >= STOP:
            nxt = EOS
        if prev in (EOS, PAD):
            nxt = PAD
        if 0 <= col < T:
            h["out"][b, col] = nxt
        h["tok"][b] = nxt
        h["pos"][b] += 1
        at = int(h["pos"][b] - s["base"][b])
        h["pos32"][b], h["seqlens"][b], h["rpos32"][b] = at, at + 1, int(h["pos"][b] + s["rope"][b])


def _logp_bound(V, big):
    """Roundings, relative to the sum of exponentials. A thread adds up at most 256 exponentials (a whole row of 2^17 tokens
    on 512 threads; a slice of 8192 on 256 threads has 32), each off by 2 (its value), and rescales its sum at most 16 times,
    3 each; the wavefront, the workgroup and the slices' join add 6 + 8 and, with a scaling of 4 each, 6 + V / 2^19 steps; the
    exponents' arguments are off by 12 big in all (5 for each term and the changes of the maximum, 2 for the reference's
    z'), the logarithm and the last subtraction by 3 (17 + 2 big)."""
    return U * (258 + 48 + 14 + 4 * (6 + V / 2 ** 19) + 51 + 18 * big)


# (B, V, columns): slices with the join, then with histories counted by token, then whole rows
CUTS = [(3, 87383, 18), (1, 87383, 18), (2, 40001, 33), (3, 87383, 2100), (5, 5463, 2100), (6, 1367, 40), (77, 5463, 24),
        (200, 33000, 18)]


@pytest.mark.parametrize("B,V,T", CUTS)
@pytest.mark.parametrize("mode", ["greedy", "gumbel", "cdf"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_steps_of_a_decode(B, V, T, mode, dt):
    temperature = 0.0 if mode == "greedy" else 0.75
    s = _problem(B, V, T, dt, B + V + T, mode == "gumbel")
    u = None if mode == "greedy" else s["u"]
    for rules in (True, False):
        d = _device(s)
        h = {k: d[k].cpu().clone() for k in STATE}
        g = torch.Generator().manual_seed(V + 1)
        for step in range(3):
            x = s["x"] if step == 0 else (3 * torch.randn(B, V, generator=g)).to(dt)
            col = h["pos"] - s["plen"]
            lens, at = col.clamp(0, T).int(), col.clamp(0, T - 1)
            kw = dict(bias=d["bias"], fallback=PAD)
            host, rows = [None, None, 1.0, 0.0, 0.0], None
            mask = torch.ones(B, V, dtype=torch.bool)
            if rules:
                rows = s["token_rows"][h["tok"]]
                kw.update(zip(("history", "lengths", "repetition", "presence", "frequency"), (d["out"].clone(), lens.to(DEV), *PENALTIES)))
                kw.update(allowed=d["allowed"], allowed_rows=rows.to(DEV))
                host = [h["out"].clone(), lens, *PENALTIES]
                mask = torch.where((rows < 0)[:, None], mask, s["masks"][rows.clamp(min=0).long()])
            now = None if u is None else u[torch.arange(B, device=DEV), at.to(DEV)].contiguous()
            want, wlogp = ops.choose_tokens(x.to(DEV), temperature=temperature, uniforms=now, **kw)
            _step(d, x.to(DEV), temperature, u, rules)
            # the choice, against the CPU's in 64 bits
            z = _rules_ref(x, *host, s["bias"], mask)
            temps = torch.full((B,), temperature)
            tok, lp, big = _choice_ref(z, temps, now.cpu() if mode == "gumbel" else None)
            zt = _tame(z) / (temperature if temperature > 0 else 1.0)
            bound = _logp_bound(V, big)
            got, glogp = want.cpu(), wlogp.cpu().double()
            none = tok < 0
            assert bool((got[none] == PAD).all()) and bool((glogp[none] == -np.inf).all())
            if mode != "cdf":
                assert torch.equal(got[~none], tok[~none])
            else:
                p = torch.softmax(zt.double(), 1)
                upto = p.cumsum(1).gather(1, got[:, None])[:, 0]
                own = p.gather(1, got[:, None])[:, 0]
                # (both the sum up to the token and the whole are off by the bound; the running sum of fp64 by less than one of it)
                assert bool(((own > 0) & (upto + 3 * bound > now.cpu()) & (upto - own - 3 * bound <= now.cpu()))[~none].all())
                lp = torch.log(own)
            assert bool(((glogp - lp).abs() <= bound)[~none].all())
            # the state
            _advance(h, s, got, wlogp.cpu(), T)
            for k in STATE:
                assert torch.equal(d[k].cpu(), h[k]), (rules, step, k)
        assert bool((d["out"].as_strided((B, 5), (T + 5, 1), d["out"].storage_offset() + T) == -3).all())


def test_the_problems_hold_what_they_are_for():
    """Every forced token happens: the tail's and the run's EOS, PAD behind the end, PAD where nothing is allowed."""
    s = _problem(77, 5463, 24, torch.float32, 77 + 5463 + 24, False)
    d = _device(s)
    _step(d, s["x"].to(DEV), 0.0, None, True)
    prev, now = s["tok"], d["tok"].cpu()
    over, tail = (prev == EOS) | (prev == PAD), s["tail"][s["tok"]]
    runs = s["run"] == STOP - 2
    assert over.any() and bool((now[over] == PAD).all()) and tail.any() and bool((now[tail] == EOS).all())
    assert runs.any() and bool((now[runs] == EOS).all())
    empty = prev == 7
    assert empty.any() and bool((now[empty] == PAD).all())
    free = ~(over | tail | runs | empty)
    assert bool((now[free] > 2).any())


@pytest.mark.parametrize("B,V,T", [(3, 87383, 18), (5, 5463, 2100), (77, 5463, 24)])
@pytest.mark.parametrize("mode", ["greedy", "gumbel", "cdf"])
def test_steps_in_a_graph(B, V, T, mode):
    """A captured step, replayed with other logits, is the eager step; eager steps of a second state in between."""
    temperature = 0.0 if mode == "greedy" else 0.75
    s = _problem(B, V, T, torch.float32, B + V + T + 1, mode == "gumbel")
    u = None if mode == "greedy" else s["u"]
    mine, twin = _device(s), _device(s)
    x = s["x"].to(DEV)
    first = {k: mine[k].clone() for k in STATE}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(mine, x, temperature, u, True)
    torch.cuda.current_stream().wait_stream(side)
    for k in STATE:
        mine[k].copy_(first[k])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(mine, x, temperature, u, True)
    g = torch.Generator(DEV).manual_seed(5)
    for _ in range(4):
        x.copy_(3 * torch.randn(B, V, generator=g, device=DEV))
        graph.replay()
        _step(twin, x, temperature, u, True)
        torch.cuda.synchronize()
        for k in STATE:
            assert torch.equal(mine[k], twin[k]), k


@pytest.mark.parametrize("T,sampling,thr", [(0.0, "inverse_cdf", 1e-2), (0.8, "gumbel", 3e-2)])
def test_engine_of_8mers(T, sampling, thr):
    """87383 tokens, two sequences: the engine's captured steps join slices; the stream against the oracle."""
    out, res, eng = run_case(k=8, T=T, steps=8, lens=(64, 31), mh=None, sampling=sampling)
    assert ops._choose_workspace(2, eng.model.tokenizer.vocab_size, 0) > 0
    check_stream(out, res, 8, thr)
