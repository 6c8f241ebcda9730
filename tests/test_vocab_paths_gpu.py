"""The paths that run the large-vocabulary operators: DecodeEngine past 512 tokens and with penalties and a grammar, the
differentiable token embedding, and a rollout, its scoring and its update together at the 6-mer vocabulary."""

import copy

import numpy as np
import pytest
import torch

from oracle import reference as R
from tests.test_engine_gpu import check_stream, gpu_copy, run_case
from viktor_amd import DecodeEngine, KmerTokenizer
from viktor_amd import gspo as G
from viktor_amd import hip_ops as ops
from viktor_amd import train as TR
from viktor_amd.synthetic import frames as synth_frames, make_model

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_greedy_stream_past_the_fused_head():
    """5-mers (1367 tokens): the engine's head, choice and state update against the oracle, in captured graphs; grouped."""
    out, res, eng = run_case(k=5, lens=(64, 200, 31), steps=14, mh=20)
    assert not eng._fused_head and eng.out.shape[0] == 3
    check_stream(out, res, 14, 1e-2)
    out, res, _ = run_case(k=5, lens=(64, 31), steps=10, mh=20, group=4)
    check_stream(out, res, 10, 1e-2)


def test_gumbel_stream_past_the_fused_head():
    out, res, _ = run_case(k=5, T=0.8, steps=12, lens=(64, 200, 31), mh=16, sampling="gumbel")
    check_stream(out, res, 12, 3e-2)


def test_inverse_cdf_stream_past_the_fused_head():
    """The uniform lies in the chosen token's interval of the oracle's running softmax sums, up to 5e-3 (the bar for
    sampled streams: how far bf16 logits move a boundary)."""
    from viktor_amd.synthetic import uniforms
    lens, steps, seed = (50, 120, 9), 12, 0
    out, res, eng = run_case(k=5, T=1.0, steps=steps, lens=lens, mh=None)
    u = uniforms(len(lens), steps, seed=seed + 2)
    out = out.cpu()
    tail = KmerTokenizer(5).tail_mask
    checked = 0
    for b in range(len(lens)):
        prev = R.BOS
        for j in range(steps):
            t = int(out[b, j])
            if prev in (R.EOS, R.PAD):
                assert t == R.PAD
            elif bool(tail[prev]):
                assert t == R.EOS
            else:
                z = res["logits"][b, j].double()
                z[[R.PAD, R.BOS]] = float("-inf")
                c = torch.softmax(z, 0).cumsum(0)
                lo = float(c[t - 1]) if t else 0.0
                assert lo - 5e-3 <= float(u[b, j]) < float(c[t]) + 5e-3, (b, j)
                checked += 1
            prev = t
    assert checked >= 6


class RuleEngine(R.RefEngine):
    """The oracle with penalties and a grammar: one sequence, its history the tokens that are fed back."""

    def __init__(self, *a, penalties=(1.0, 0.0, 0.0), grammar=None, fed=None, **k):
        super().__init__(*a, **k)
        self.pen, self.grammar, self.fed, self.step = penalties, grammar, fed, 0

    def _choose(self, logits, prev, run, u):
        z = logits.float().clone()
        rep, pres, freq = self.pen
        for v, c in zip(*torch.unique(self.fed[:self.step], return_counts=True)):
            x = z[v] / rep if z[v] > 0 else z[v] * rep
            z[v] = x - freq * c - pres
        if self.grammar is not None:
            mask, rows = self.grammar
            if rows[prev] >= 0:
                z = torch.where(mask[rows[prev]], z, torch.full_like(z, float("-inf")))
        self.step += 1
        return super()._choose(z, prev, run, u)


@pytest.mark.parametrize("k,T,group", [(1, 0.0, 1), (1, 0.9, 1), (5, 0.0, 1), (1, 0.0, 2)])
def test_penalties_and_grammar_stream(k, T, group):
    """Penalties over the tokens produced so far and masks by the previous token, against the oracle: no base twice in a
    row (k = 1), nothing but even ids after an odd one (k = 5)."""
    lens, steps, pen = [40, 130, 75], 18, (1.3, 0.4, 0.2)
    m = make_model(k, n_layers=2, seed=5, norm_jitter=0.1, bias_jitter=0.1)
    V = m.tokenizer.vocab_size
    if k == 1:
        mask = torch.ones(4, V, dtype=torch.bool)
        mask[torch.arange(4), torch.arange(3, 7)] = False
        rows = torch.tensor([-1, -1, -1, 0, 1, 2, 3])
    else:
        mask = (torch.arange(V) % 2 == 0)[None]
        rows = torch.where(torch.arange(V) % 2 == 1, 0, -1)
    fr = synth_frames(1, sum(lens), 512, seed=6)[0]
    wins = [w for w in fr.split(lens) for _ in range(group)]
    all_lens = [w.shape[0] for w in wins]
    u = torch.rand(len(wins), steps, V, generator=torch.Generator().manual_seed(7))
    eng = DecodeEngine(gpu_copy(m), len(wins), steps, max(lens), temperature=T, max_homopolymer=None, sampling="gumbel",
                       group_size=group, repetition_penalty=pen[0], presence_penalty=pen[1], frequency_penalty=pen[2],
                       grammar=(mask, rows))
    bias = torch.zeros(V)
    bias[[R.PAD, R.BOS, R.EOS]] = float("-inf")
    eng.bias.copy_(bias)
    if T > 0:
        eng.set_uniforms(u.to(DEV))
    out = eng.generate(torch.cat(wins).to(DEV), all_lens, steps=steps).clone().cpu()
    ref = R.RefModel(m, "fused")
    for b, w in enumerate(wins):
        oracle = RuleEngine(ref, steps, temperature=T, max_homopolymer=None, bias=bias, sampling="gumbel", penalties=pen,
                            grammar=(mask, rows), fed=out[b])
        res = oracle.run([w], uniforms=u[b:b + 1] if T > 0 else None, forced=out[b:b + 1])
        check_stream(out[b:b + 1], res, steps, 3e-2 if T > 0 else 1e-2)
    if k == 1:
        assert not bool((out[:, 1:] == out[:, :-1]).any())


def test_rules_in_graphs_equal_eager_and_neutral_rules_change_nothing():
    """Captured steps equal eager ones bit for bit; at 7 tokens a grammar that allows everything gives the plain engine's
    stream (its head a product of its own)."""
    m = make_model(1, n_layers=2, seed=8, norm_jitter=0.1)
    lens, steps = [60, 33], 20
    fr = synth_frames(1, sum(lens), 512, seed=9)[0].to(DEV)
    outs = []
    for graph in (True, False):
        eng = DecodeEngine(gpu_copy(m), 2, steps, 60, cuda_graph=graph, check_every=4, repetition_penalty=1.2,
                           frequency_penalty=0.1, logprobs=True, max_homopolymer=None)
        out = eng.generate(fr, lens, steps=steps).clone()
        outs.append((out, eng.logp.clone()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    every = (torch.ones(1, 7, dtype=torch.bool), torch.zeros(7, dtype=torch.long))
    plain = DecodeEngine(gpu_copy(m), 2, steps, 60, logprobs=True)
    ruled = DecodeEngine(gpu_copy(m), 2, steps, 60, logprobs=True, grammar=every)
    a, b = plain.generate(fr, lens, steps=steps).clone(), ruled.generate(fr, lens, steps=steps).clone()
    assert torch.equal(a, b)
    assert float((plain.logp - ruled.logp).abs().max()) < 1e-3


def test_engine_refuses_bad_rules():
    m = gpu_copy(make_model(1, n_layers=1, seed=1))
    ok = torch.ones(2, 7, dtype=torch.bool)
    for kw in ({"repetition_penalty": 0.0}, {"grammar": (ok.int(), torch.zeros(7, dtype=torch.long))},
               {"grammar": (ok[:, :6], torch.zeros(7, dtype=torch.long))}, {"grammar": (ok, torch.full((7,), 2))},
               {"grammar": (ok, torch.zeros(6, dtype=torch.long))}, {"grammar": (ok, torch.zeros(7))}):
        with pytest.raises(ValueError):
            DecodeEngine(m, 2, 8, 16, cuda_graph=False, **kw)


@pytest.mark.parametrize("V,d,wt", [(343, 512, torch.float32), (1367, 512, torch.float32), (5463, 64, torch.bfloat16), (50, 30, torch.float32),
                                    (1367, 24, torch.float16)])
@pytest.mark.parametrize("scale,pad", [(1.0, None), (22.627417, 0)])
def test_token_embedding(V, d, wt, scale, pad):
    """Forward exact; the gradient within the roundings of fp32 sums (an id's rows in sequence at most, the product, and the
    weight's own type), on either side of the sorted gradient's border, with a batch of ids and a broadcast gradient."""
    g = torch.Generator().manual_seed(V)
    w = torch.randn(V, d, generator=g).to(wt).to(DEV).requires_grad_()
    tok = torch.randint(0, V, (7, 33), generator=g)
    tok[:, 20:] = 0
    y = TR.token_embedding(w, tok.to(DEV), scale, pad)
    assert y.dtype == torch.float32 and torch.equal(y.detach(), w.detach().float()[tok.to(DEV)] * scale)
    L = torch.randn(7, 33, d, generator=g)
    (y * L.to(DEV)).sum().backward()
    keep = tok.reshape(-1) != (-1 if pad is None else pad)
    want = torch.zeros(V, d, dtype=torch.float64)
    mag = torch.zeros_like(want)
    rows = L.reshape(-1, d).double()
    want.index_add_(0, tok.reshape(-1)[keep], rows[keep])
    mag.index_add_(0, tok.reshape(-1)[keep], rows[keep].abs())
    tol = 2.0 ** -24 * (7 * 33 + 3) * scale * mag + torch.finfo(wt).eps / 2 * want.abs() * scale
    assert w.grad.dtype == wt and bool(((w.grad.cpu().double() - want * scale).abs() <= tol * 1.01).all())
    w.grad = None
    TR.token_embedding(w, tok.to(DEV), scale, pad).sum().backward()  # (an expanded gradient)
    count = torch.zeros(V, dtype=torch.float64).index_add_(0, tok.reshape(-1)[keep], torch.ones(int(keep.sum()), dtype=torch.float64))
    assert torch.allclose(w.grad.cpu().double(), (count * scale)[:, None].expand(V, d), rtol=2 ** -8 if wt != torch.float32 else 2 ** -22, atol=0)


@pytest.mark.parametrize("V", [343, 5463])
def test_token_embedding_in_a_graph(V):
    """Forward and backward captured together, replayed with other ids and gradients, eager calls in between."""
    g = torch.Generator().manual_seed(V)
    w = torch.randn(V, 64, generator=g).to(DEV).requires_grad_()
    tok, L = torch.zeros(6000, dtype=torch.long, device=DEV), torch.zeros(6000, 64, device=DEV)

    def call():
        y = TR.token_embedding(w, tok, 2.0, 0)
        return y.detach(), torch.autograd.grad(y, w, L)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        tok.copy_(torch.randint(0, V, (6000,), generator=g))
        L.copy_(torch.randn(6000, 64, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


def test_rollout_scoring_and_update_of_6mers():
    """A model of the 6-mer vocabulary (5463 tokens) through the public path: sampled rollout with penalties, its
    log-probabilities against the scoring forward's, rewards, one update; the embedding's gradient is the one that the
    small vocabularies' kernel gives on the same rows."""
    k, n_win, group, P = 6, 2, 4, 96
    model = make_model(k, n_layers=2, seed=21, norm_jitter=0.1).to(DEV)
    inf = G.bf16_copy(model)
    fr = synth_frames(n_win, P, 512, seed=22).to(DEV)
    plens = torch.tensor([P, P - 17], device=DEV)
    eng = G.engine(inf, n_win * group, temperature=1.0, max_frames=P, max_new_tokens=24, group_size=group, sampling="gumbel",
                   logprobs=True, repetition_penalty=1.1, frequency_penalty=0.1)
    torch.manual_seed(23)
    calls, ended = G.decode(eng, fr.repeat_interleave(group, 0), plens.repeat_interleave(group), model.tokenizer)
    assert len(calls) == n_win * group and any(len(c) > 0 for c in calls)
    lp, mask = G.token_logprobs(model, fr.repeat_interleave(group, 0), plens.repeat_interleave(group), calls, ended)
    assert bool(torch.isfinite(lp[mask.to(DEV)]).all())
    # scored without penalties: the first token's is the engine's own (its history is empty), up to the bf16 of the logits
    # (a step of 2^-6 at sizes up to 4 on each side) and the bf16 inference copy
    first = [b for b in range(len(calls)) if len(calls[b]) >= k]
    assert first and max(abs(float(lp[b, 0] - eng.logp[b, 0])) for b in first) < 0.1
    seen = {}
    real = ops.embed_grad_sorted

    def both(d_rows, tokens, vocab, **kw):
        seen["diff"] = (real(d_rows, tokens, vocab, **kw) - ops.embed_grad(d_rows, tokens, vocab)).abs().max()
        seen["size"] = ops.embed_grad(d_rows.abs(), tokens, vocab).max()
        return real(d_rows, tokens, vocab, **kw)

    before = model.decoder.embed.weight.detach().clone()
    opt = TR.HipAdamW(list(model.parameters()), lr=1e-4)
    reward = np.random.default_rng(3).random((n_win, group))
    ops.embed_grad_sorted = both
    try:
        st = TR.gspo_update(model, opt, fr, plens, calls, ended, reward, group, updates=1, micro=group)
    finally:
        ops.embed_grad_sorted = real
    assert st["n"] == n_win * group and np.isfinite(st["grad_norm"][0]) and st["grad_norm"][0] > 0
    assert float(seen["diff"]) <= 2.0 ** -24 * 600 * float(seen["size"])
    assert not torch.equal(before, model.decoder.embed.weight.detach())
    G.sync(inf, model)
    again, _ = G.decode(eng, fr.repeat_interleave(group, 0), plens.repeat_interleave(group), model.tokenizer)
    assert len(again) == n_win * group
