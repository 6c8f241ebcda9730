"""The operators of large vocabularies -- embed_lookup, embed_grad_sorted, process_logits, choose_tokens -- against plain
implementations on the CPU: fp64 sums for the gradient, fp32 steps in the documented order for the rules (bit for bit),
fp64 scores for the choice. Tolerances count roundings: 2^-24 relative per fp32 operation."""

import numpy as np
import pytest
import torch

from viktor_amd import hip_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
F32 = torch.float32
U = 2.0 ** -24  # half a step of fp32, relative


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same(a, b):
    """Equal values, NaN where NaN."""
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---- lookup --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [1, 3, 7, 8, 64, 65, 130, 511, 512, 1000, 1025])
@pytest.mark.parametrize("wt,ot", [(F32, F32), (F32, BF), (BF, F32), (BF, BF)])
def test_embed_lookup(d, wt, ot):
    """Equal to the fp32 product rounded once, at every row count around the wavefronts' groups; ids outside the table
    (past 32 bits too) give zero rows."""
    g = _gen(d)
    V, scale = 1367, 22.627417
    w = torch.randn(V, d, generator=g).to(wt)
    for n in (1, 15, 16, 17, 65, 259):
        tok = torch.randint(0, V, (n,), generator=g)
        tok[0] = V - 1
        bad = torch.zeros(n, dtype=torch.bool)
        if n > 8:
            tok[[1, 3, 5]] = torch.tensor([-1, V, 2 ** 32 + 4])
            bad[[1, 3, 5]] = True
        want = (w.float()[tok.clamp(0, V - 1).where(~bad, torch.zeros_like(tok))] * scale).to(ot)
        want[bad] = 0
        assert _same(ops.embed_lookup(w.to(DEV), tok.to(DEV), scale=scale, out_dtype=ot), want), n


def test_embed_lookup_shapes():
    w = torch.randn(343, 512, generator=_gen(1))
    tok = torch.randint(0, 343, (3, 5), generator=_gen(2))
    got = ops.embed_lookup(w.to(DEV), tok.to(DEV))
    assert got.shape == (3, 5, 512) and _same(got, w[tok])
    assert ops.embed_lookup(w.to(DEV), tok[:0].to(DEV)).shape == (0, 5, 512)


def test_embed_lookup_of_more_rows_than_a_launch():
    """2^24 workgroups of 16 rows and some: the rows behind the first launch, and those around its end."""
    n, V = 2 ** 28 + 37, 343
    w = torch.randn(V, 1, generator=_gen(1)).to(BF).to(DEV)
    tok = torch.arange(n, device=DEV) % (V + 1)  # (one id past the table)
    got = ops.embed_lookup(w, tok).view(-1)
    for a in range(0, n, 2 ** 26):
        t = tok[a:a + 2 ** 26]
        assert torch.equal(got[a:a + 2 ** 26], torch.where(t < V, w[:, 0][t.clamp(max=V - 1)], 0.0)), a


# ---- gradient --------------------------------------------------------------------------------------------------------------

def _grad_ref(rows, tok, V, scale, pad=None):
    """(fp64 gradient, what an element may be off by, in units of U): a run's sum is at most 127 additions in a chunk (of up
    to 64 positions) and the next; a longer one's 64 in each chunk, its chunks' sums over 32 groups, and the groups; then one
    product. Chunks of 16 (n <= 16384) and 32 (n <= 102400) have fewer additions each and no more in all:
    16 + 16384 / 512 + 32 and 32 + 102400 / 1024 + 32 are below 127 and 127 + 102400 / 2048."""
    keep = (tok >= 0) & (tok < V) & (tok != (-1 if pad is None else pad))
    out = torch.zeros(V, rows.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    out.index_add_(0, tok[keep], rows[keep].double())
    mag.index_add_(0, tok[keep], rows[keep].double().abs())
    adds = 127 + len(tok) / (64 * 32) + 1 + 32 + 2
    return out * scale, adds * U * mag * abs(scale)


def _check_grad(got, ref, what=""):
    want, tol = ref
    assert bool(((got.cpu().double() - want).abs() <= tol).all()), (what, float((got.cpu().double() - want).abs().max()))


def _ids(kind, n, V, g):
    if kind == "skew":
        return (torch.rand(n, generator=g).pow(3) * V).long().clamp(max=V - 1)
    if kind == "one":
        return torch.full((n,), V // 2, dtype=torch.long)
    if kind == "padded":
        t = torch.randint(0, V, (n,), generator=g)
        t[torch.rand(n, generator=g) < 0.4] = 0
        return t
    return torch.randint(0, V, (n,), generator=g)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 193, 1003, 4095, 4096, 4097, 8192, 8193, 20001])
@pytest.mark.parametrize("kind", ["flat", "skew", "one", "padded"])
def test_embed_grad_sorted(n, kind):
    """Both sorts, chunk and tile borders, and tokens that a large part of the rows share."""
    for V, d, dt in ((1, 64, F32), (7, 5, BF), (511, 128, BF), (512, 33, F32), (5463, 512, F32)):
        g = _gen(n + V)
        tok = _ids(kind, n, V, g)
        rows = torch.randn(n, d, generator=g).to(dt)
        got = ops.embed_grad_sorted(rows.to(DEV), tok.to(DEV), V, scale=1.5)
        _check_grad(got, _grad_ref(rows, tok, V, 1.5), (V, d))


@pytest.mark.parametrize("d", [1, 3, 4, 6, 63, 64, 65, 127, 128, 129, 255, 256, 260, 511, 513, 700, 768, 769, 1000, 1024, 1030, 2050])
@pytest.mark.parametrize("dt", [F32, BF])
def test_embed_grad_sorted_widths(d, dt):
    g = _gen(d)
    n, V = 700, 37
    tok = _ids("padded", n, V, g)
    rows = torch.randn(n, d, generator=g).to(dt)
    _check_grad(ops.embed_grad_sorted(rows.to(DEV), tok.to(DEV), V), _grad_ref(rows, tok, V, 1.0))


@pytest.mark.parametrize("V", [87383, 262143, 262144, 300001])
def test_embed_grad_sorted_vocabularies(V):
    """Two and three radix passes; the last id."""
    g = _gen(V)
    n, d = 9000, 16
    tok = _ids("skew", n, V, g)
    tok[[5, 700, 8999]] = V - 1
    rows = torch.randn(n, d, generator=g)
    _check_grad(ops.embed_grad_sorted(rows.to(DEV), tok.to(DEV), V), _grad_ref(rows, tok, V, 1.0))


@pytest.mark.parametrize("n", [300, 9000])
def test_embed_grad_sorted_ignores_and_accumulates(n):
    """Ids outside the table and the padding id add nothing (whatever their rows hold); a strided view of the rows; added to
    a table, rows without ids left as they were."""
    g = _gen(n)
    V, d = 1367, 64
    tok = _ids("skew", n, V // 2, g)
    wide = torch.randn(n, 96, generator=g)
    bad = torch.rand(n, generator=g) < 0.3
    bad[0] = bad[n - 1] = True
    tok[bad] = torch.tensor([-1, V, 2 ** 40, 5])[torch.randint(0, 4, (int(bad.sum()),), generator=g)]
    wide[(tok < 0) | (tok >= V) | (tok == 5)] = float("nan")
    rows = wide[:, 8:8 + d]
    ref = _grad_ref(rows, tok, V, 0.5, pad=5)
    dev_rows = wide.to(DEV)[:, 8:8 + d]
    got = ops.embed_grad_sorted(dev_rows, tok.to(DEV), V, scale=0.5, pad=5)
    _check_grad(got, ref)
    old = torch.randn(V, d, generator=g)
    table = old.to(DEV)
    back = ops.embed_grad_sorted(dev_rows, tok.to(DEV), V, scale=0.5, pad=5, out=table, accumulate=True)
    assert back is table
    want = old.double() + ref[0]
    tol = ref[1] + 2 * U * (old.double().abs() + ref[0].abs())
    assert bool(((table.cpu().double() - want).abs() <= tol).all())
    used = torch.zeros(V, dtype=torch.bool)
    used[tok[(tok >= 0) & (tok < V) & (tok != 5)]] = True
    assert torch.equal(table.cpu()[~used], old[~used])


@pytest.mark.parametrize("lens", [(64, 64, 64), (63, 65, 64), (1, 64, 127, 1), (1, 128, 63), (64, 128, 64), (65, 63, 200, 5),
                                  (130, 1, 1, 190), (10, 54, 64, 64, 64, 10), (63, 129, 63, 129, 1), (500,), (32, 300, 40, 300)])
@pytest.mark.parametrize("ignored", [0, 70])
def test_embed_grad_sorted_run_lengths(lens, ignored):
    """Runs of given lengths against the chunks of 64 positions: ending and starting at borders, one past them, holding a
    whole chunk or two, with ignored rows behind the last; shuffled, by both sorts."""
    for more in (0, 5000):  # (past the counting sort: one more long run at the end)
        V = 20
        tok = torch.cat([torch.full((m,), 2 * i, dtype=torch.long) for i, m in enumerate((*lens, more))])
        tok = torch.cat([tok, torch.full((ignored,), -1, dtype=torch.long)])
        tok = torch.cat([tok, torch.full((ignored,), V + 5, dtype=torch.long)]) if more else tok
        g = _gen(sum(lens) + more)
        tok = tok[torch.randperm(len(tok), generator=g)]
        rows = torch.randn(len(tok), 260, generator=g)
        _check_grad(ops.embed_grad_sorted(rows.to(DEV), tok.to(DEV), V), _grad_ref(rows, tok, V, 1.0), more)


@pytest.mark.parametrize("chunk,n", [(16, 2000), (16, 16384), (32, 16385), (32, 102400), (64, 102401), (64, 131073)])
@pytest.mark.parametrize("dt", [F32, BF])
def test_embed_grad_sorted_run_borders(chunk, n, dt):
    """Runs that end and start at, before and behind the borders of chunks of each size, among runs of a few rows, the last
    chunk's included; added to a table too."""
    c = chunk
    g = _gen(n)
    V, d = 3 * n // 4, 12
    for lens in ((c, c, c), (c - 1, c + 1, c), (1, c, 2 * c - 1, 1), (c, 2 * c, c), (c + 1, c - 1, 3 * c + 8, 5), (2 * c + 2, 1, 1, 3 * c - 2),
                 (c - 1, 2 * c + 1, c - 1, 2 * c + 1, 1), (40 * c + 3,), (c // 2, 5 * c, c // 2, 5 * c)):
        ends = torch.cat([torch.full((m,), i, dtype=torch.long) for i, m in enumerate(lens)])
        tok = torch.cat([ends, V - 1 - ends, torch.randint(20, V - 20, (n - 2 * len(ends),), generator=g)])
        tok = tok[torch.randperm(n, generator=g)]
        rows = torch.randn(n, d, generator=g).to(dt)
        ref = _grad_ref(rows, tok, V, 2.0)
        _check_grad(ops.embed_grad_sorted(rows.to(DEV), tok.to(DEV), V, scale=2.0), ref, lens)
        table = torch.ones(V, d, device=DEV)
        ops.embed_grad_sorted(rows.to(DEV), tok.to(DEV), V, scale=2.0, out=table, accumulate=True)
        _check_grad(table, (ref[0] + 1, ref[1] + 2 * U * (ref[0].abs() + 1)), lens)


def test_embed_grad_sorted_many_tiles():
    """More tiles than a scatter sums itself (524288 rows): the scan in its own launch; a run of a third of the rows."""
    n, V, d = 524288 + 8193, 5463, 8
    g = _gen(9)
    tok = _ids("skew", n, V, g)
    tok[torch.rand(n, generator=g) < 0.33] = 17
    rows = torch.randn(n, d, generator=g)
    _check_grad(ops.embed_grad_sorted(rows.to(DEV), tok.to(DEV), V), _grad_ref(rows, tok, V, 1.0))


def test_embed_grad_sorted_of_nothing():
    none = torch.zeros(0, dtype=torch.long, device=DEV)
    assert not ops.embed_grad_sorted(torch.zeros(0, 64, device=DEV), none, 100).any()
    tok = torch.full((50,), -3, dtype=torch.long, device=DEV)
    assert not ops.embed_grad_sorted(torch.ones(50, 64, device=DEV), tok, 100).any()


def test_embed_grad_sorted_twice_the_same_bits():
    g = _gen(11)
    tok = _ids("padded", 30000, 5463, g).to(DEV)
    rows = torch.randn(30000, 512, generator=g).to(DEV)
    a = ops.embed_grad_sorted(rows, tok, 5463)
    for _ in range(3):
        assert torch.equal(ops.embed_grad_sorted(rows, tok, 5463), a)


def test_embedding_gradient_against_differences():
    """sum(L * lookup(W)) is linear in W: its derivative along a direction is the gradient's product with it."""
    g = _gen(3)
    V, d, n = 200, 32, 500
    w, dw = torch.randn(V, d, generator=g), torch.randn(V, d, generator=g)
    tok, L = torch.randint(0, V, (n,), generator=g), torch.randn(n, d, generator=g)

    def f(t):
        return float((ops.embed_lookup(t.to(DEV), tok.to(DEV), scale=2.0).cpu().double() * L.double()).sum())

    grad = ops.embed_grad_sorted(L.to(DEV), tok.to(DEV), V, scale=2.0).cpu().double()
    slope = (f(w + dw) - f(w - dw)) / 2
    size = 2.0 * float((L.abs().double() * (w.abs() + dw.abs())[tok].double()).sum())
    assert abs(slope - float((grad * dw.double()).sum())) <= 90 * U * size


# ---- rules on logits -------------------------------------------------------------------------------------------------------

def _rules_ref(x, hist=None, lens=None, rep=1.0, pres=0.0, freq=0.0, bias=None, mask=None):
    """fp32 on the CPU, one rounding per step. mask: bool [B, V]."""
    z = x.float().clone()
    B, V = z.shape
    col = lambda t: (t if torch.is_tensor(t) else torch.full((B,), t)).float()[:, None]  # noqa: E731
    if hist is not None:
        count = torch.zeros(B, V)
        for b in range(B):
            for t in hist[b, :max(0, min(int(lens[b]), hist.shape[1]))].tolist():
                if 0 <= t < V:
                    count[b, t] += 1
        seen = count > 0
        z = torch.where(seen, torch.where(z > 0, z / col(rep), z * col(rep)), z)
        z = torch.where(seen, z - col(freq) * count, z)
        z = torch.where(seen, z - col(pres), z)
    if bias is not None:
        z = z + bias
    if mask is not None:
        z = torch.where(mask, z, torch.full_like(z, float("-inf")))
    return z


def _case(B, V, T, seed, dt=F32):
    g = _gen(seed)
    x = (3 * torch.randn(B, V, generator=g)).to(dt)
    hist = (torch.rand(B, T, generator=g).pow(3) * V).long().clamp(max=V - 1)
    lens = torch.randint(0, T + 1, (B,), generator=g).int()
    rep = 1 + 0.5 * torch.rand(B, generator=g)
    pres, freq = torch.rand(B, generator=g), 0.3 * torch.rand(B, generator=g)
    bias = torch.randn(V, generator=g)
    bias[0] = float("-inf")
    masks = torch.rand(3, V, generator=g) < 0.5
    masks[:, V - 1] = True
    rows = torch.randint(-1, 3, (B,), generator=g).int()
    mask = torch.where((rows < 0)[:, None], torch.ones(1, V, dtype=torch.bool), masks[rows.clamp(min=0).long()])
    return x, hist, lens, rep, pres, freq, bias, masks, rows, mask


def _dev(*ts):
    return [t.to(DEV) for t in ts]


SIZES = [(1, 1, 1), (3, 7, 5), (2, 343, 40), (5, 1367, 100), (4, 5463, 300), (2, 2049, 2049), (600, 33, 9), (512, 9001, 20), (3, 40001, 500)]


@pytest.mark.parametrize("B,V,T", SIZES)
@pytest.mark.parametrize("dt,odt", [(F32, F32), (BF, BF), (BF, F32), (F32, BF)])
def test_process_logits(B, V, T, dt, odt):
    x, hist, lens, rep, pres, freq, bias, masks, rows, mask = _case(B, V, T, B + V, dt)
    want = _rules_ref(x, hist, lens, rep, pres, freq, bias, mask)
    kw = dict(zip(("history", "lengths", "repetition", "presence", "frequency", "bias"), _dev(hist, lens, rep, pres, freq, bias)))
    packed = ops.pack_allowed(masks).to(DEV)
    got = ops.process_logits(x.to(DEV), **kw, allowed=packed, allowed_rows=rows.to(DEV), out_dtype=odt)
    assert _same(got, want.to(odt))


def test_process_logits_parts():
    """Each rule alone, scalars for penalties, one mask row for all or one per sequence, a bias per sequence, in place, a
    strided view in and out with the columns around it left as they were."""
    B, V, T = 4, 1367, 60
    x, hist, lens, rep, pres, freq, bias, masks, rows, mask = _case(B, V, T, 5)
    dx, dh, dl = _dev(x, hist, lens)
    assert _same(ops.process_logits(dx), x)
    for kw in ({"rep": 1.3}, {"pres": 0.7}, {"freq": 0.2}, {"pres": -0.5, "freq": -0.1}, {"rep": 0.7}):
        names = {"rep": "repetition", "pres": "presence", "freq": "frequency"}
        f = {k: float(np.float32(v)) for k, v in kw.items()}
        got = ops.process_logits(dx, dh, dl, **{names[k]: v for k, v in f.items()})
        assert _same(got, _rules_ref(x, hist, lens, **f)), kw
    biases = torch.randn(B, V, generator=_gen(6))
    assert _same(ops.process_logits(dx, bias=biases.to(DEV)), _rules_ref(x, bias=biases))
    assert _same(ops.process_logits(dx, allowed=ops.pack_allowed(masks[:1]).to(DEV)), _rules_ref(x, mask=masks[:1].expand(B, V)))
    each = torch.rand(B, V, generator=_gen(7)) < 0.5
    assert _same(ops.process_logits(dx, allowed=ops.pack_allowed(each).to(DEV)), _rules_ref(x, mask=each))
    want = _rules_ref(x, hist, lens, rep, pres, freq, bias, mask)
    args = dict(history=dh, lengths=dl, repetition=rep.to(DEV), presence=pres.to(DEV), frequency=freq.to(DEV),
                bias=bias.to(DEV), allowed=ops.pack_allowed(masks).to(DEV), allowed_rows=rows.to(DEV))
    mine = dx.clone()
    assert ops.process_logits(mine, **args, out=mine) is mine and _same(mine, want)
    wide_in, wide_out = torch.zeros(B, V + 9, device=DEV), torch.full((B, V + 13), 7.0, device=DEV)
    wide_in[:, 3:3 + V] = dx
    ops.process_logits(wide_in[:, 3:3 + V], **args, out=wide_out[:, 5:5 + V])
    assert _same(wide_out[:, 5:5 + V], want)
    assert bool((wide_out[:, :5] == 7).all()) and bool((wide_out[:, 5 + V:] == 7).all())
    assert ops.process_logits(dx[:0]).shape == (0, V)


def test_process_logits_odd_values():
    """NaN and infinities: kept where allowed, gone where masked; history lengths outside 0 .. T and ids outside the
    vocabulary (past 32 bits too) are taken as documented; a token that fills the whole history."""
    V, T = 4099, 300
    x = torch.randn(5, V, generator=_gen(1))
    x[:, 10], x[:, 11], x[:, 12] = float("nan"), float("inf"), float("-inf")
    mask = torch.ones(5, V, dtype=torch.bool)
    mask[1, 10:13] = False
    mask[2] = False
    hist = torch.randint(0, V, (5, T), generator=_gen(2))
    hist[0, :50] = torch.tensor([-1, V, 2 ** 32 + 7, -2 ** 40, 2 ** 31] * 10)
    hist[3] = 77
    hist[4, :4] = torch.tensor([10, 11, 12, 10])
    lens = torch.tensor([T, -5, T + 1000, T, 4], dtype=torch.int32)
    want = _rules_ref(x, hist, lens, 1.25, 0.5, 0.25, None, mask)
    dx, dh, dl = _dev(x, hist, lens)
    got = ops.process_logits(dx, dh, dl, 1.25, 0.5, 0.25, allowed=ops.pack_allowed(mask).to(DEV))
    assert _same(got, want)
    assert bool((got[2] == float("-inf")).all())


def test_process_logits_longest_history():
    """65535 times one token: the largest count."""
    V, T = 100, 65535
    x = torch.randn(2, V, generator=_gen(1))
    hist = torch.full((2, T), 41, dtype=torch.long)
    hist[1, ::2] = 40
    lens = torch.tensor([T, T], dtype=torch.int32)
    got = ops.process_logits(*_dev(x, hist, lens), frequency=0.001)
    c = torch.zeros(2, V)
    c[0, 41], c[1, 40], c[1, 41] = T, (T + 1) // 2, T // 2
    assert _same(got, x - torch.tensor(0.001) * c)


# ---- choice ----------------------------------------------------------------------------------------------------------------

def _tame(z):
    return torch.nan_to_num(z, nan=float("-inf"), posinf=torch.finfo(F32).max, neginf=float("-inf"))


def _choice_ref(z, temp=None, u=None):
    """(token, logp fp64, greatest |z'|) of fp32 logits after the rules; temp fp32 [B] or None; u [B, V] or None."""
    z = _tame(z)
    if temp is not None:
        z = torch.where(temp[:, None] > 0, z / torch.where(temp > 0, temp, torch.ones_like(temp))[:, None], z)
    s = z.double()
    if u is not None:
        noise = -torch.log(-torch.log(u.double().clamp(min=1e-20)))
        s = torch.where((temp > 0)[:, None] & (s > float("-inf")), s + noise, s)
    best = s.max(1, keepdim=True).values
    V = z.shape[1]
    tok = torch.where(s == best, torch.arange(V), V).min(1).values
    none = best[:, 0] == float("-inf")
    zd = z.double() - z.double().max(1, keepdim=True).values.clamp(min=-3e38)  # (before any sum: 3e38 + 0.7 is 3e38)
    lp = zd.gather(1, tok.clamp(max=V - 1)[:, None])[:, 0] - torch.log(torch.exp(zd).sum(1))
    big = torch.where(z.abs() < 3e38, z.abs(), torch.zeros_like(z)).max(1).values.double()
    return torch.where(none, -1, tok), torch.where(none, torch.full_like(lp, float("-inf")), lp), big


def _check_logp(got, want, big):
    """Roundings, relative to the sum of exponentials: each term's argument (z' and its product with log2 e: 3 |z'|, the
    size of z' - m at most 2 |z'|) and value (2), a thread's up to 64 additions with as many changes of the maximum, the
    joins (16), the logarithm and the last two subtractions (6 |z'| and the log's size, at most 12)."""
    got, inf = got.cpu().double(), want == float("-inf")
    assert bool((got[inf] == float("-inf")).all())
    assert bool(((got - want).abs()[~inf] <= U * (200 + 16 * big)[~inf]).all()), float((got - want).abs()[~inf].max())


@pytest.mark.parametrize("B,V,T", SIZES)
@pytest.mark.parametrize("dt", [F32, BF])
def test_choose_tokens_greedy(B, V, T, dt):
    """bf16 logits tie often: the lowest id wins."""
    x, hist, lens, rep, pres, freq, bias, masks, rows, mask = _case(B, V, T, B + V + 1, dt)
    tok, lp, big = _choice_ref(_rules_ref(x, hist, lens, rep, pres, freq, bias, mask))
    kw = dict(zip(("history", "lengths", "repetition", "presence", "frequency", "bias"), _dev(hist, lens, rep, pres, freq, bias)))
    got, glp = ops.choose_tokens(x.to(DEV), **kw, allowed=ops.pack_allowed(masks).to(DEV), allowed_rows=rows.to(DEV), fallback=-1)
    assert torch.equal(got.cpu(), tok)
    _check_logp(glp, lp, big)


@pytest.mark.parametrize("B,V,T", SIZES)
@pytest.mark.parametrize("dt", [F32, BF])
def test_choose_tokens_gumbel(B, V, T, dt):
    """The fp64 scores' choice, rows of temperature 0 (greedy) and uniforms of 0 among them."""
    x, hist, lens, rep, pres, freq, bias, masks, rows, mask = _case(B, V, T, B + V + 2, dt)
    g = _gen(V)
    temp = 0.5 + torch.rand(B, generator=g)
    temp[::3] = 0
    u = torch.rand(B, V, generator=g)
    u[:, ::5] = 0
    tok, lp, big = _choice_ref(_rules_ref(x, hist, lens, rep, pres, freq, bias, mask), temp, u)
    kw = dict(zip(("history", "lengths", "repetition", "presence", "frequency", "bias"), _dev(hist, lens, rep, pres, freq, bias)))
    got, glp = ops.choose_tokens(x.to(DEV), **kw, allowed=ops.pack_allowed(masks).to(DEV), allowed_rows=rows.to(DEV),
                                 temperature=temp.to(DEV), uniforms=u.to(DEV), fallback=-1)
    assert torch.equal(got.cpu(), tok)
    _check_logp(glp, lp, big)


def test_choose_tokens_gumbel_near_ties():
    """Scores that fp32 cannot tell apart: equal logits under uniforms one step apart, in every place of the vocabulary."""
    V = 3001
    u = torch.full((64, V), 0.3)
    a = torch.randint(0, V, (64,), generator=_gen(1))
    b = (a + torch.randint(1, V, (64,), generator=_gen(2))) % V
    near = torch.tensor(0.9999)
    up = torch.nextafter(near, torch.tensor(1.0))
    u[torch.arange(64), a], u[torch.arange(64), b] = near, up
    x = torch.full((64, V), 0.25)
    got, _ = ops.choose_tokens(x.to(DEV), temperature=0.7, uniforms=u.to(DEV))
    assert torch.equal(got.cpu(), b)
    u[torch.arange(64), b] = near
    got, _ = ops.choose_tokens(x.to(DEV), temperature=0.7, uniforms=u.to(DEV))
    assert torch.equal(got.cpu(), torch.minimum(a, b))


def _check_cdf(z, temp, u, got, glp):
    B = len(u)
    greedy, glpref, big = _choice_ref(z, temp)
    zt = torch.where(temp[:, None] > 0, z / torch.where(temp > 0, temp, torch.ones_like(temp))[:, None], z)
    for b in range(B):
        if greedy[b] < 0 or temp[b] <= 0:
            assert got[b] == greedy[b]
            continue
        p = torch.softmax(zt[b].double(), 0)
        c = p.cumsum(0)
        t = int(got[b])
        tol = 2 * U * float(200 + 16 * big[b])
        assert p[t] > 0 and float(c[t]) + tol > float(u[b]) >= float(c[t] - p[t]) - tol, b
        _check_logp(glp[b:b + 1], torch.log(p[t:t + 1]), big[b:b + 1])


@pytest.mark.parametrize("B,V,T", SIZES)
@pytest.mark.parametrize("dt", [F32, BF])
def test_choose_tokens_inverse_cdf(B, V, T, dt):
    """u lies in the chosen token's interval of the fp64 running softmax sums, up to the roundings that the
    log-probability counts too (both the sum up to it and the whole)."""
    x, hist, lens, rep, pres, freq, bias, masks, rows, mask = _case(B, V, T, B + V + 3, dt)
    g = _gen(V + 1)
    temp = 0.5 + torch.rand(B, generator=g)
    u = torch.rand(B, generator=g)
    u[0] = 0
    if B > 1:
        temp[1] = 0
    z = _tame(_rules_ref(x, hist, lens, rep, pres, freq, bias, mask))
    kw = dict(zip(("history", "lengths", "repetition", "presence", "frequency", "bias"), _dev(hist, lens, rep, pres, freq, bias)))
    got, glp = ops.choose_tokens(x.to(DEV), **kw, allowed=ops.pack_allowed(masks).to(DEV), allowed_rows=rows.to(DEV),
                                 temperature=temp.to(DEV), uniforms=u.to(DEV), fallback=-1)
    got, glp = got.cpu(), glp.cpu()
    _check_cdf(z, temp, u, got, glp)


@pytest.mark.parametrize("B,V,T", [(192, 70001, 300), (250, 20000, 2048), (300, 40000, 64), (2, 600001, 500)])
@pytest.mark.parametrize("dt", [F32, BF])
def test_choose_tokens_inverse_cdf_of_long_rows(B, V, T, dt):
    """Rows of several batches in one workgroup, and of many slices: every target from the first token with weight to the
    last, most of a row's weight on tokens of its history in some, rows without anything."""
    x, hist, lens, rep, pres, freq, bias, masks, rows, mask = _case(B, V, T, B + V + 4, dt)
    g = _gen(V + 2)
    heavy = torch.arange(0, B, 3)
    x[heavy[:, None], hist[heavy, :5].clamp(max=V - 1)] = torch.tensor(14.0, dtype=dt)
    temp = 0.7 + torch.rand(B, generator=g)
    temp[4::9] = 0
    u = torch.rand(B, generator=g)
    u[::5] = 0
    u[1::5] = 1 - 2.0 ** -24
    x[7::50] = float("-inf")
    z = _tame(_rules_ref(x, hist, lens, rep, pres, freq, bias, mask))
    kw = dict(zip(("history", "lengths", "repetition", "presence", "frequency", "bias"), _dev(hist, lens, rep, pres, freq, bias)))
    args = dict(**kw, allowed=ops.pack_allowed(masks).to(DEV), allowed_rows=rows.to(DEV), temperature=temp.to(DEV),
                uniforms=u.to(DEV), fallback=-1)
    got, glp = ops.choose_tokens(x.to(DEV), **args)
    _check_cdf(z, temp, u, got.cpu(), glp.cpu())
    again = ops.choose_tokens(x.to(DEV), **args)
    assert torch.equal(again[0], got) and torch.equal(again[1], glp)


def test_choose_tokens_odd_values():
    """NaN never wins, +inf counts as the largest value (the lower id of two), masked infinities are nothing, a row without
    anything gives the fallback and -inf; uniforms at 1 - 2^-24."""
    V = 5000
    x = torch.randn(6, V, generator=_gen(4))
    x[0, [5, 4000]] = float("nan")
    x[1, [4321, 17]] = float("inf")
    x[2] = float("-inf")
    x[3] = float("nan")
    x[4, 100] = float("inf")
    mask = torch.ones(6, V, dtype=torch.bool)
    mask[4, 100] = False
    mask[5] = False
    packed = ops.pack_allowed(mask).to(DEV)
    tok, lp, big = _choice_ref(_rules_ref(x, mask=mask))
    tok = torch.where(tok < 0, 2, tok)
    got, glp = ops.choose_tokens(x.to(DEV), allowed=packed, fallback=2)
    assert torch.equal(got.cpu(), tok) and got[1] == 17 and got[5] == 2
    _check_logp(glp, lp, big)
    assert abs(float(glp[1]) + float(np.log(2))) < 1e-6
    for u in (torch.full((6,), 1 - 2.0 ** -24), torch.zeros(6)):
        got, glp = ops.choose_tokens(x.to(DEV), allowed=packed, temperature=1.0, uniforms=u.to(DEV), fallback=2)
        ok = _tame(_rules_ref(x, mask=mask))
        for b in (0, 1, 4):
            assert ok[b, int(got[b])] > float("-inf") and not bool(x[b, int(got[b])].isnan())
        assert got[1] in (17, 4321) and got[2] == got[3] == got[5] == 2
    u = torch.rand(6, V, generator=_gen(5))
    tok, lp, big = _choice_ref(_rules_ref(x, mask=mask), torch.full((6,), 0.8), u)
    got, glp = ops.choose_tokens(x.to(DEV), allowed=packed, temperature=0.8, uniforms=u.to(DEV), fallback=-1)
    assert torch.equal(got.cpu()[[0, 2, 3, 4, 5]], tok[[0, 2, 3, 4, 5]]) and got[1] in (17, 4321)


def test_choose_tokens_lowest_values_and_extreme_temperatures():
    """A row of the type's lowest value everywhere, where z / T leaves fp32's range: its tokens are alike, and the first
    allowed one is taken (noise below fp64's resolution there); the inverse CDF takes any. Tiny temperatures order by z,
    an infinite one by the noise alone. In one launch, in slices, and with a history among the tokens."""
    for V in (40, 5000, 40001):
        low = torch.full((3, V), torch.finfo(F32).min)
        mask = torch.ones(3, V, dtype=torch.bool)
        mask[1, :7] = False
        mask[2] = False
        u = torch.rand(3, V, generator=_gen(V))
        hist, n = torch.full((3, 2), 20), torch.full((3,), 2, dtype=torch.int32)
        logv = np.log([V, V - 7])
        packed = ops.pack_allowed(mask).to(DEV)
        for T in (0.5, 1e-30):
            got, lp = ops.choose_tokens(low.to(DEV), *_dev(hist, n), frequency=1.0, allowed=packed, temperature=T,
                                        uniforms=u.to(DEV), fallback=-1)
            assert got.tolist() == [0, 7, -1], (V, T)
            _check_logp(lp, torch.tensor([-logv[0], -logv[1], -np.inf]), torch.zeros(3))
            got, lp = ops.choose_tokens(low.to(DEV), allowed=packed, temperature=T, uniforms=u[:, 0].contiguous().to(DEV), fallback=-1)
            assert 0 <= got[0] and 7 <= got[1] < V and got[2] == -1
            _check_logp(lp, torch.tensor([-logv[0], -logv[1], -np.inf]), torch.zeros(3))
        x = torch.randn(3, V, generator=_gen(V + 1))
        for z in (x, x - 100):  # scores past the range on either side
            for T in (1e-38, 1e-44):
                got, lp = ops.choose_tokens(z.to(DEV), allowed=packed, temperature=T, uniforms=u.to(DEV), fallback=-1)
                want = torch.where(mask, z, torch.tensor(-np.inf)).max(1).indices
                want[2] = -1
                assert torch.equal(got.cpu(), want), (V, T)
                assert lp[:2].tolist() == [0, 0]
        got, lp = ops.choose_tokens(x.to(DEV), allowed=packed, temperature=float("inf"), uniforms=u.to(DEV), fallback=-1)
        want = torch.where(mask, u, torch.tensor(-1.0)).max(1).indices
        want[2] = -1
        assert torch.equal(got.cpu(), want)
        _check_logp(lp, torch.tensor([-logv[0], -logv[1], -np.inf]), torch.zeros(3))
        temps = torch.full((3,), float("inf")).to(DEV)
        got, lp = ops.choose_tokens(x.to(DEV), allowed=packed, temperature=temps, uniforms=u[:, 0].contiguous().to(DEV), fallback=-1)
        assert 0 <= got[0] < V and 7 <= got[1] < V and got[2] == -1
        _check_logp(lp, torch.tensor([-logv[0], -logv[1], -np.inf]), torch.zeros(3))


def test_choose_tokens_of_the_widest_whole_rows():
    """512 rows of 2^17 tokens with the longest hashed history, the largest shared memory of one launch: six rows checked."""
    B, V, T = 512, 2 ** 17, 2048
    g = torch.Generator(DEV).manual_seed(1)
    x = (3 * torch.randn(B, V, generator=g, device=DEV)).to(BF)
    hist = (torch.rand(B, T, generator=g, device=DEV).pow(3) * V).long().clamp(max=V - 1)
    lens = torch.full((B,), T, dtype=torch.int32, device=DEV)
    u = torch.rand(B, V, generator=g, device=DEV)
    rows = [0, 1, 255, 256, 300, 511]
    z = _rules_ref(x[rows].cpu(), hist[rows].cpu(), lens[rows].cpu(), 1.25, 0.5, 0.25)
    for temp in (0.0, 0.75):
        t = torch.full((B,), temp, device=DEV)
        tok, lp, big = _choice_ref(z, t[rows].cpu(), u[rows].cpu())
        got, glp = ops.choose_tokens(x, hist, lens, 1.25, 0.5, 0.25, temperature=t if temp else 0.0, uniforms=u if temp else None)
        assert torch.equal(got[rows].cpu(), tok)
        _check_logp(glp[rows], lp, big)


@pytest.mark.parametrize("B,V,T", [(40, 1367, 2000), (200, 5463, 2048), (9, 21847, 3000), (3, 87383, 2048), (200, 87383, 700)])
def test_choose_tokens_again_the_same_bits(B, V, T):
    """Long histories, whose tokens are found in another order each time: tokens and log-probabilities stay."""
    x, hist, lens, rep, pres, freq, bias, masks, rows, mask = _case(B, V, T, B + V + 5)
    x, hist, lens, rep, pres, freq, bias, rows = _dev(x, hist, lens, rep, pres, freq, bias, rows)
    u = torch.rand(B, V, generator=torch.Generator(DEV).manual_seed(6), device=DEV)
    allowed = ops.pack_allowed(masks).to(DEV)
    for kw in ({}, {"temperature": 0.9, "uniforms": u}, {"temperature": 0.9, "uniforms": u[:, 0].contiguous()}):
        first = ops.choose_tokens(x, hist, lens, rep, pres, freq, bias, allowed, rows, **kw)
        for _ in range(6):
            again = ops.choose_tokens(x, hist, lens, rep, pres, freq, bias, allowed, rows, **kw)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1]), list(kw)


# ---- streams, graphs, refusals -----------------------------------------------------------------------------------------------

def test_vocabulary_ops_in_a_graph():
    """Captured together, replayed with other inputs of the same shapes, eager calls and a second graph in between."""
    V, d, n, B = 5463, 64, 5000, 9
    g = _gen(8)

    def inputs():
        return (torch.randn(V, d, generator=g), torch.randint(0, V, (n,), generator=g), torch.randn(n, d, generator=g),
                torch.randn(B, V, generator=g), torch.randint(0, V, (B, 50), generator=g), torch.rand(B, V, generator=g))

    w, tok, rows, z, hist, u = _dev(*inputs())
    lens = torch.full((B,), 50, dtype=torch.int32, device=DEV)

    def call():
        return (ops.embed_lookup(w, tok, scale=2.0), ops.embed_grad_sorted(rows, tok, V, pad=3),
                ops.process_logits(z, hist, lens, 1.2, 0.1, 0.1), *ops.choose_tokens(z, hist, lens, 1.2),
                *ops.choose_tokens(z, hist, lens, 1.2, temperature=0.9, uniforms=u))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            eager = call()  # on another stream than the inputs'
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, call()):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for _ in range(3):
        for t, new in zip((w, tok, rows, z, hist, u), inputs()):
            t.copy_(new)
        for graph, _ in graphs:
            graph.replay()
        want = call()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_vocabulary_ops_side_by_side():
    """Calls of two streams at once, each with workspaces of its own."""
    V, d, n, B = 21847, 64, 30000, 40
    g = torch.Generator(DEV).manual_seed(3)
    sets = []
    for _ in range(2):
        sets.append((torch.randint(0, V, (n,), generator=g, device=DEV), torch.randn(n, d, generator=g, device=DEV),
                     torch.randn(B, V, generator=g, device=DEV), torch.rand(B, V, generator=g, device=DEV)))

    def call(tok, rows, z, u):
        return (ops.embed_grad_sorted(rows, tok, V), *ops.choose_tokens(z), *ops.choose_tokens(z, temperature=0.9, uniforms=u),
                *ops.choose_tokens(z, temperature=0.9, uniforms=u[:, 0].contiguous()))

    want = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


def test_process_logits_out_beside_logits():
    """Columns of one buffer as logits and out; views that share elements are refused."""
    B, V = 5, 1367
    buf = torch.randn(B, 2 * V + 3, generator=_gen(1)).to(DEV)
    want = buf[:, :V] + 1
    bias = torch.ones(V, device=DEV)
    ops.process_logits(buf[:, :V], bias=bias, out=buf[:, V + 3:])
    assert torch.equal(buf[:, V + 3:], want)
    flat = torch.zeros(2 * B * V, device=DEV)
    z = flat[:B * V].view(B, V)
    ops.process_logits(z, bias=bias, out=flat[B * V:].view(B, V))
    assert bool((flat[B * V:] == 1).all()) and not bool(flat[:B * V].any())
    for out in (buf[:, 1:1 + V], buf[:, V - 1:2 * V - 1]):
        with pytest.raises(AssertionError):
            ops.process_logits(buf[:, :V], out=out)
    for out in (flat[4:4 + B * V].view(B, V), flat[V:V + B * V].view(B, V), flat.view(BF)[2:2 + B * V].view(B, V)):
        with pytest.raises(AssertionError):
            ops.process_logits(z, out=out)
    with pytest.raises(ops._lib.HipLibraryError):
        ops.process_logits(z, out=flat.view(BF)[:B * V].view(B, V))


def test_vocabulary_ops_refuse():
    z = torch.zeros(3, 40, device=DEV)
    h, n = torch.zeros(3, 5, dtype=torch.long, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    w, tok = torch.zeros(40, 8, device=DEV), torch.zeros(6, dtype=torch.long, device=DEV)
    rows = torch.zeros(6, 8, device=DEV)
    m = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    bad = [
        lambda: ops.embed_lookup(w.half(), tok), lambda: ops.embed_lookup(w, tok.int()), lambda: ops.embed_lookup(w.t(), tok),
        lambda: ops.embed_lookup(w, tok, out_dtype=torch.float16),
        lambda: ops.embed_grad_sorted(rows, tok[:5], 40), lambda: ops.embed_grad_sorted(rows.t(), tok, 40),
        lambda: ops.embed_grad_sorted(rows, tok, 0), lambda: ops.embed_grad_sorted(rows, tok, 2 ** 32 + 40), lambda: ops.embed_grad_sorted(rows, tok, 40, accumulate=True),
        lambda: ops.embed_grad_sorted(rows, tok, 40, out=torch.zeros(40, 9, device=DEV)),
        lambda: ops.embed_grad_sorted(rows[:1].expand(6, 8), tok, 40),
        lambda: ops.process_logits(z.half()), lambda: ops.process_logits(z, repetition=1.1),
        lambda: ops.process_logits(z, h, None, 1.1), lambda: ops.process_logits(z, h, n.long(), 1.1),
        lambda: ops.process_logits(z, h, n, 0.0), lambda: ops.process_logits(z, h.int(), n, 1.1),
        lambda: ops.process_logits(z, bias=torch.zeros(39, device=DEV)), lambda: ops.process_logits(z, allowed=m[:2]),
        lambda: ops.process_logits(z, allowed=m[:, :1]), lambda: ops.process_logits(z, allowed_rows=n),
        lambda: ops.process_logits(z, out=torch.zeros(3, 40, dtype=torch.float16, device=DEV)),
        lambda: ops.process_logits(z[:1].expand(3, 40)),
        lambda: ops.choose_tokens(torch.empty(1, 2 ** 30 + 1, dtype=BF, device=DEV)),
        lambda: ops.choose_tokens(z, temperature=0.5), lambda: ops.choose_tokens(z, temperature=torch.ones(3, device=DEV)),
        lambda: ops.choose_tokens(z, uniforms=torch.zeros(3, 39, device=DEV)),
        lambda: ops.choose_tokens(z, uniforms=torch.zeros(3, 40, dtype=BF, device=DEV)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError):
            f()
            print("not refused:", i)
    with pytest.raises(ops._lib.HipLibraryError):
        ops.process_logits(z, torch.zeros(3, 65536, dtype=torch.long, device=DEV), n, 1.1)
