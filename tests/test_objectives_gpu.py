"""The objectives on logits and the teacher's lists against their definitions in 64 bits (tests/objectives_plain.py)."""

import math

import pytest
import torch
import torch.utils.checkpoint

from viktor_amd import hip_ops as ops, objectives

from . import objectives_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def logits_of(B, T, V, dtype, seed, sure=True, layout="plain"):
    """Logits with a fairly sure target each, the targets, and a mask whose sequences end at different lengths (the first
    one full, the second one empty)."""
    g = torch.Generator(DEV).manual_seed(seed)
    y = torch.randint(0, V, (B, T), generator=g, device=DEV)
    z = 2 * torch.randn(B, T, V, generator=g, device=DEV)
    if sure:
        z.scatter_add_(2, y[..., None], (math.log(V) + 3 * torch.rand(B, T, 1, generator=g, device=DEV)))
    z = z.to(dtype)
    ends = torch.randint(0, T + 1, (B, 1), generator=g, device=DEV)
    ends[0] = T
    if B > 1:
        ends[1] = 0
    mask = torch.arange(T, device=DEV) < ends
    if layout == "sliced":        # rows of a longer sequence, off 16 bytes
        big = torch.zeros(B, T + 3, V + 5, dtype=dtype, device=DEV)
        big[:, 2:T + 2, 3:V + 3] = z
        z = big[:, 2:T + 2, 3:V + 3]
    elif layout == "turned":      # token-major
        z = z.transpose(0, 1).contiguous().transpose(0, 1)
    return z, y, mask, g


def near(got, want, tol, what):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & (got != want)  # (equal infinities)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - want).abs().max()))


def check_gradient(got, z, loss, dtype, lp_tol, what):
    want = torch.autograd.grad(loss, z)[0]
    # a row's coefficient: its largest gradient is at least c (1 - 1 / V) of it but for a row sure of its target; bounded by
    # the sum of the row's parts on either side
    coef = want.abs().sum(-1, keepdim=True) + want.abs().amax()
    assert got.dtype == dtype
    near(got, want, plain.gradient_tolerance(want, coef, dtype, lp_tol), what + ": gradient")


FORMS = [1, 2, 7, 8, 13, 16, 33, 127, 343, 385, 500, 1367, 1537, 2500, 5463, 8191, 12289, 21847, 22600, 45100, 60001]
LONG = [87383, 90200, 180300, 250001]


def policy_inputs(B, T, V, dtype, seed, layout="plain", far=0.3):
    z, y, mask, g = logits_of(B, T, V, dtype, seed, layout=layout)
    lp = torch.log_softmax(z.double(), -1).gather(2, y[..., None])[..., 0].float()
    old = lp + far * torch.randn(B, T, generator=g, device=DEV)
    ref = lp + far * torch.randn(B, T, generator=g, device=DEV)
    return z, y, mask, old, ref, g


def check_policy(z, y, mask, old, adv, ref, **kw):
    """All outputs of policy_score. Away from the clip's borders: tokens within 1e-4 of one (float lp decides there) are
    masked out for both."""
    V, dtype = z.shape[2], z.dtype
    on = plain.counting(y, mask, V)
    lp0 = torch.log_softmax(torch.where(on[..., None], z.double(), 0.0), -1).gather(2, y.clamp(0, V - 1)[..., None])[..., 0]
    r = torch.exp(lp0 - old.double())
    lo, hi = 1 - kw.get("eps_lo", 0.2), 1 + kw.get("eps_hi", 0.2)
    mask = mask & ~(((r - lo).abs() < 1e-4) | ((r - hi).abs() < 1e-4))
    got = ops.policy_score(z, y, mask, old, adv, ref, **kw)
    leaf, want = plain.policy(z, y, mask, old, adv, ref, **kw)
    tol = plain.lp_tolerance(z[on] if bool(on.any()) else z.new_zeros(1), V)
    near(got["lp"], want["lp"], tol, "lp")
    # d pg / d lp = -r A (or 0), d kl / d lp = 1 - exp(x): lp's error times those, and a rounding of each
    a = (adv[:, None] if adv.dim() == 1 else adv).double().abs()
    u = 2.0 ** -22
    r = torch.where(on, r, 0.0)
    near(got["pg"], want["pg"], (tol + u) * (r + 1) * a + 1e-30, "pg")
    if ref is not None:
        x = torch.where(on, ref.double() - lp0, 0.0)
        near(got["kl"], want["kl"], tol * (x.exp() - 1).abs() + tol ** 2 + u * want["kl"].abs() + 1e-30, "kl")
    else:
        assert got["kl"] is None
    size = float((want["pg"].abs() + (0 if ref is None else abs(kw.get("kl_coef", 0)) * want["kl"].abs())).detach().amax()) if y.numel() else 0.0
    near(got["loss"], want["loss"], (8 * tol + u) * max(size, 1e-6) * (1.0 if kw.get("per") != "token" or kw.get("inv_n") is None
                                                                     else kw["inv_n"] * y.numel()) + 8 * tol, "loss")
    # (the coefficient -r A - beta (exp(x) - 1) is off by lp's error times its own derivative)
    x = None if ref is None else (torch.where(on, ref.double() - lp0, 0.0)).exp()
    scale = 1 + float((r * a).max() if y.numel() else 0) + (0 if ref is None else float(x.max()))
    check_gradient(got["dlogits"], leaf, want["loss"], dtype, 4 * tol * scale, "policy")
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", FORMS)
def test_policy_vocabularies(V, dtype):
    B, T = (5, 9) if V < 20000 else (3, 4)
    z, y, mask, old, ref, g = policy_inputs(B, T, V, dtype, V)
    adv = torch.randn(B, generator=g, device=DEV)
    check_policy(z, y, mask, old, adv, ref, kl_coef=0.05, eps_hi=0.28)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", LONG)
def test_policy_long_rows(V, dtype):
    z, y, mask, old, ref, g = policy_inputs(3, 2, V, dtype, V, layout="sliced")
    check_policy(z, y, mask, old, torch.randn(3, 2, generator=g, device=DEV), ref, kl_coef=0.05, per="token")


@pytest.mark.parametrize("B,T", [(1, 1), (1, 300), (300, 1), (7, 130), (64, 33)])
@pytest.mark.parametrize("V", [7, 343, 5463])
def test_policy_batches(B, T, V):
    for k, (per, inv_n, with_ref) in enumerate([("sequence", None, True), ("token", None, False), ("sequence", 0.01, False),
                                                ("token", 0.002, True)]):
        z, y, mask, old, ref, g = policy_inputs(B, T, V, (BF16, F32)[k % 2], 31 * B + T + k)
        adv = torch.randn((B,) if k < 2 else (B, T), generator=g, device=DEV)
        check_policy(z, y, mask, old, adv, ref if with_ref else None, kl_coef=0.1 if with_ref else 0.0, per=per, inv_n=inv_n)


@pytest.mark.parametrize("layout", ["sliced", "turned"])
@pytest.mark.parametrize("V", [7, 343, 1367, 5463])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_policy_layouts(V, layout, dtype):
    z, y, mask, old, ref, g = policy_inputs(4, 6, V, dtype, 5, layout)
    assert not z.is_contiguous()
    check_policy(z, y, mask, old, torch.randn(4, generator=g, device=DEV), ref, kl_coef=0.02)


@pytest.mark.parametrize("V", [7, 343, 5463, 25000])
def test_policy_what_does_not_count_is_not_looked_at(V):
    """NaN and infinities in masked tokens' logits, old_lp and ref_lp, targets outside the vocabulary; a mask that leaves
    nothing at all."""
    z, y, mask, old, ref, g = policy_inputs(5, 8, V, F32, 3)
    y[0, 1], y[0, 2], y[0, 3] = -1, V, 2 ** 40
    y[1] = -5
    on = plain.counting(y, mask, V)
    for bad in (math.nan, math.inf, -math.inf):
        z2 = torch.where(on[..., None], z, bad)
        old2, ref2 = torch.where(on, old, bad), torch.where(on, ref, bad)
        got = check_policy(z2, y, mask, old2, torch.randn(5, generator=g, device=DEV), ref2, kl_coef=0.3)
        assert bool((got["dlogits"][~on] == 0).all()) and bool((got["lp"][~on] == 0).all())
    none = ops.policy_score(z2, y, torch.zeros_like(mask), old2, torch.full((5,), math.nan, device=DEV), ref2, kl_coef=0.3,
                            per="token")
    assert float(none["loss"]) == 0 and bool((none["dlogits"] == 0).all()) and bool((none["kl"] == 0).all())


def test_policy_masked_vocabulary_entries():
    """-inf and the type's lowest value among a counting row's logits: probability and gradient 0 there."""
    for low in (-math.inf, torch.finfo(BF16).min):
        z, y, mask, old, ref, g = policy_inputs(3, 5, 343, BF16, 4)
        z[..., 100:300] = low
        z.scatter_(2, y[..., None], 3.0)
        lp = torch.log_softmax(z.double(), -1).gather(2, y[..., None])[..., 0].float()
        got = ops.policy_score(z, y, mask, lp - 0.05, torch.ones(3, device=DEV))
        leaf, want = plain.policy(torch.where(z < -1e30, -1e30, z.double()), y, mask, lp - 0.05, torch.ones(3, device=DEV))
        near(got["lp"], want["lp"], plain.lp_tolerance(z[z > -1e30], 343), "lp")
        check_gradient(got["dlogits"], leaf, want["loss"], BF16, 8 * plain.lp_tolerance(z[z > -1e30], 343), "masked entries")


@pytest.mark.parametrize("V", [20, 343])
def test_policy_of_far_and_impossible_tokens(V):
    """A target's logit far below the row's maximum, or -inf: the ratio exp(lp - old_lp) keeps its 32 bits down to the type's
    smallest numbers and is 0 at last; a reference policy that rules a token out has an infinite kl with a finite slope."""
    B, T = 2, 8
    z, _, _, g = logits_of(B, T, V, F32, 77, sure=False)
    y = torch.randint(0, V, (B, T), generator=g, device=DEV)
    mask = torch.ones(B, T, dtype=torch.bool, device=DEV)
    far = torch.tensor([0.0, -12.0, -25.0, -45.0, -80.0, -70.0, -700.0, -math.inf], device=DEV)
    z = z.scatter(2, y[..., None], (z.gather(2, y[..., None])[..., 0] + far)[..., None])
    old = torch.full((B, T), -3.0, device=DEV)
    adv = torch.tensor([1.0, -2.0], device=DEV)
    _, want = plain.policy(z, y, mask, old, adv)
    got = ops.policy_score(z, y, mask, old, adv)
    assert bool(torch.isfinite(got["loss"])) and not bool(got["dlogits"].isnan().any())
    assert bool(((got["lp"] == -math.inf) == (far == -math.inf)).all())
    # the ratio's error: that of lp, 5e-7 of the sum's logarithm in 32-bit terms at most, and 2^-24 of its rounding
    inner = want["pg"][0, :7].abs() > 1e-37
    off = ((got["pg"][0, :7] - want["pg"][0, :7]).abs() / want["pg"][0, :7].abs().clamp(min=1e-300))[inner]
    assert bool((off < 1e-6).all())
    # the gradient: c (onehot - p), c = A r / n below the clip's border for A > 0, 0 for A < 0 (the clip's side is the lesser)
    lp = torch.log_softmax(z.double(), -1)
    c = (torch.exp(lp.gather(2, y[..., None])[..., 0] + 3.0) * 1.0 / (B * T))[0, 1:]
    one = torch.nn.functional.one_hot(y, V).double()
    grad = -c[:, None] * (one - lp.exp())[0, 1:]
    # (p: |z - top| < 24 rounded to 32 bits twice, 2^-24 of 24 and 0.69 of 2^-24 of 35, 2.9e-6; c and the exponential, 6e-7)
    assert bool(((got["dlogits"][0, 1:].double() - grad).abs() <= 4e-6 * grad.abs() + 1e-37).all())
    assert not bool(got["dlogits"][1, 1:].any())
    ref = torch.full((B, T), -math.inf, device=DEV)
    ref[:, 4:] = -3.0
    got = ops.policy_score(z[:, :6].contiguous(), y[:, :6].contiguous(), mask[:, :6], old[:, :6], adv * 0, ref[:, :6], kl_coef=0.5)
    x = ref[:, :6].double() - lp.gather(2, y[..., None])[:, :6, 0]
    c = 0.5 * -torch.expm1(x) / (B * 6)
    grad = c[..., None] * (one - lp.exp())[:, :6]
    assert bool((got["kl"][:, :4] == math.inf).all()) and float(got["loss"]) == math.inf
    assert bool(((got["dlogits"].double() - grad).abs() <= 4e-6 * grad.abs() + 1e-37).all())


@pytest.mark.parametrize("V", [7, 20, 343, 5463, 21847, 87383, 250001])
def test_gradient_of_rows_sure_of_their_target(V):
    """c (1 - p) where p is next to 1 keeps its 32 bits, in the policy's gradient and in the pairs'."""
    B, T = 2, 5
    z, y, _, g = logits_of(B, T, V, F32, 79, sure=False)
    mask = torch.ones(B, T, dtype=torch.bool, device=DEV)
    z = z.clamp(-9, 9).scatter(2, y[..., None], 20.0)
    lp = torch.log_softmax(z.double(), -1).gather(2, y[..., None])[..., 0]
    old = lp.float()
    adv = torch.tensor([1.0, -2.0], device=DEV)
    zp, want = plain.policy(z, y, mask, old, adv, eps_lo=0.3, eps_hi=0.3)
    zq, pairs = plain.preference(z, y, mask)
    for got, leaf, loss in ((ops.policy_score(z, y, mask, old, adv, eps_lo=0.3, eps_hi=0.3), zp, want["loss"]),
                            (ops.preference_score(z, y, mask), zq, pairs["loss"])):
        grad = torch.autograd.grad(loss, leaf)[0].gather(2, y[..., None])
        # (the others' exponentials: |z - top| < 30 rounded to 32 bits, and 0.69 of 43; c, 1 / s and the products: 2.7e-6)
        off = (got["dlogits"].gather(2, y[..., None]).double() - grad).abs()
        assert bool((grad != 0).all()) and bool((off <= 4e-6 * grad.abs()).all()), float((off / grad.abs()).max())


@pytest.mark.parametrize("V", [7, 20, 343, 5463, 21847, 87383])
def test_exponentials_far_below_the_top(V):
    """A row of one logit t above all others: 1 - p is the others' exponentials alone, and so is the target's gradient."""
    T = 128
    z = torch.zeros(1, T, V, device=DEV)
    z[0, :, 3] = 10 + torch.arange(T, device=DEV) * 0.109375  # (differences without a rounding)
    y = torch.full((1, T), 3, device=DEV)
    mask = torch.ones(1, T, dtype=torch.bool, device=DEV)
    old = torch.log_softmax(z.double(), -1)[..., 3].float()
    adv = torch.ones(1, device=DEV)
    # 1 - p without the cancellation of p in 64 bits: 2^-53 is 4e-7 of the six others' 2.8e-10
    rest = (V - 1) * torch.exp(-z[0, :, 3].double())
    grad = -torch.exp(-torch.log1p(rest) - old[0].double()) * rest / (1 + rest) / T
    off = ((ops.policy_score(z, y, mask, old, adv)["dlogits"][0, :, 3].double() - grad) / grad).abs()
    # an exponential's ulp 1.2e-7, log 2 in 32 bits 7e-8, six roundings of 2^-24; and what the others' sum loses in one of 64
    # bits that the top's 1 is part of: 2^-53 with each addition behind it, V or a thread's 176 and the group's 16 at most
    assert bool((off <= 6e-7 + min(V, 192) * 2.0 ** -53 / rest).all()), float(off.max())


def test_policy_clip_and_its_borders():
    """Ratios of exactly 1, inside, and past each border with both signs: clipped tokens have no gradient from the
    objective. Two logits, where log-probabilities are known."""
    z = torch.zeros(1, 6, 2, device=DEV)
    y = torch.zeros(1, 6, dtype=torch.long, device=DEV)
    lp = math.log(0.5)
    old = lp - torch.log(torch.tensor([[1.0, 1.1, 1.5, 1.5, 0.5, 0.5]], device=DEV))
    adv = torch.tensor([[2.0, -1.0, 1.0, -1.0, 1.0, -1.0]], device=DEV)
    got = ops.policy_score(z, y, torch.ones(1, 6, dtype=torch.bool, device=DEV), old, adv, per="token", inv_n=1.0)
    want_pg = torch.tensor([[-2.0, 1.1, -1.2, 1.5, -0.5, 0.8]], device=DEV)
    near(got["pg"], want_pg, 1e-6, "pg")
    g = torch.tensor([[-2.0, 1.1, 0.0, 1.5, -0.5, 0.0]], device=DEV)
    near(got["dlogits"], g[..., None] * torch.tensor([0.5, -0.5], device=DEV), 1e-6, "gradient")


def test_policy_kl_without_cancellation():
    """Log-ratios of 1e-7 to 60: kl relative to 64 bits on the same lp (two logits, lp exact to 1e-8)."""
    x = torch.tensor([[1e-7, -1e-5, 1e-3, -0.03, 0.4999, -0.5001, 2.0, -20.0, 60.0]], device=DEV)
    T = x.shape[1]
    z = torch.zeros(1, T, 2, device=DEV)
    y = torch.zeros(1, T, dtype=torch.long, device=DEV)
    ref = (math.log(0.5) + x.double()).float()
    got = ops.policy_score(z, y, torch.ones(1, T, dtype=torch.bool, device=DEV), ref, torch.zeros(1, device=DEV), ref)
    x64 = ref.double() - math.log(0.5)
    want = torch.expm1(x64) - x64
    # lp is off by 3e-8 (the logarithm's) and its derivative is 1 - exp(x); then one rounding
    near(got["kl"], want, 4e-8 * torch.expm1(x64).abs() + 2e-15 + 2.0 ** -23 * want, "kl")


# ---- preference ---------------------------------------------------------------------------------------------------------

def check_preference(z, y, mask, ref, scale=1.0, **kw):
    V, T = z.shape[2], z.shape[1]
    got = ops.preference_score(z, y, mask, ref, **kw)
    leaf, want = plain.preference(z, y, mask, ref, **kw)
    on = plain.counting(y, mask, V)
    tol = plain.lp_tolerance(z[on] if bool(on.any()) else z.new_zeros(1), V)
    near(got["lp"], want["lp"], tol, "lp")
    # a margin is beta times a difference of sums of T log-ratios, each off by lp's error and a rounding of the ratio
    reach = float((want["lp"] - (0 if ref is None else torch.where(on, ref, 0.0))).detach().abs().max()) if y.numel() else 0.0
    beta = kw.get("beta", 0.1)
    mtol = beta * 2 * T * (tol + 2.0 ** -24 * reach) / scale + 2.0 ** -23 * (want["margin"].abs() + 1)
    near(got["margin"], want["margin"], mtol, "margin")
    P = max(want["margin"].numel(), 1)
    times = kw["inv_n"] * P if kw.get("inv_n") else 1.0
    m = float(mtol.detach().max()) if want["margin"].numel() else 0.0
    near(got["loss"], want["loss"], times * m + 2.0 ** -23 * (1 + float(want["loss"].detach().abs())), "loss")
    # a sequence's coefficient: the slopes of its pairs (each off by m / 4) with beta / P / length
    check_gradient(got["dlogits"], leaf, want["loss"], z.dtype, 4 * tol + m, "preference")
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", FORMS + LONG[:2])
def test_preference_vocabularies(V, dtype):
    B, T = (6, 7) if V < 20000 else (2, 3)
    z, y, mask, old, ref, g = policy_inputs(B, T, V, dtype, V + 1)
    check_preference(z, y, mask, ref, beta=0.3)


@pytest.mark.parametrize("B,T", [(2, 1), (2, 400), (40, 3), (10, 66)])
@pytest.mark.parametrize("V", [7, 343, 5463])
def test_preference_pairs(B, T, V):
    """Pairs of any sequences: in several pairs, in none, the same twice, outside the batch; lengths, smoothing, target."""
    z, y, mask, old, ref, g = policy_inputs(B, T, V, F32, B + T)
    pairs = torch.randint(0, B, (3 * B, 2), generator=g, device=DEV)
    pairs[0] = pairs[1]
    pairs[2] = 0
    pairs[3] = torch.tensor([B, 0], device=DEV)
    pairs[4] = torch.tensor([0, -1], device=DEV)
    pairs[5, 0] = 2 ** 40
    lengths = torch.randint(1, 50, (B,), generator=g, device=DEV).float()
    for kw in ({}, {"smoothing": 0.2, "target": 0.5}, {"lengths": lengths, "beta": 2.0, "inv_n": 0.01},
               {"lengths": lengths, "smoothing": 1.0}):
        got = check_preference(z, y, mask, ref, pairs=pairs, **kw)
        assert float(got["margin"][3]) == 0 and float(got["margin"][4]) == 0
    check_preference(z, y, mask, None, pairs=pairs[:1])
    one = ops.preference_score(z, y, mask, ref, pairs=pairs[:0])
    assert float(one["loss"]) == 0 and one["margin"].shape == (0,) and bool((one["dlogits"] == 0).all())


@pytest.mark.parametrize("B,T,P", [(64, 5, 1024), (64, 5, 1025), (66, 5, 40), (200, 50, 900), (2, 8192, 3), (2, 8193, 3)])
def test_preference_both_ways_of_the_pairs(B, T, P):
    """The pairs in one workgroup and in three launches, on both sides of the borders between them."""
    z, y, mask, old, ref, g = policy_inputs(B, T, 20, F32, B + P, far=0.05)
    pairs = torch.randint(0, B, (P, 2), generator=g, device=DEV)
    check_preference(z, y, mask, ref, pairs=pairs, beta=0.05)
    check_preference(z, y, mask, ref, beta=0.05, lengths=1 + torch.rand(B, generator=g, device=DEV))


def test_preference_of_impossible_calls():
    """A call with a token of probability 0 has a log-ratio of -inf: its pair's margin is infinite, and the loss of a pair that
    is as sure as that on the right side is 0 without smoothing, infinite with it."""
    z, y, _, _ = logits_of(4, 6, 343, BF16, 78)
    mask = torch.ones(4, 6, dtype=torch.bool, device=DEV)
    for call, smoothing, loss in ((1, 0.0, None), (1, 0.1, math.inf), (0, 0.0, math.inf), (0, 1.0, None), (1, 1.0, math.inf)):
        x = z.clone()
        x[call, 2, y[call, 2]] = -math.inf
        got = ops.preference_score(x, y, mask, smoothing=smoothing)
        assert got["margin"][0] == (math.inf if call else -math.inf)
        _, want = plain.preference(z[2:], y[2:], mask[2:], smoothing=smoothing)
        if loss is None:  # the other pair's alone
            near(got["loss"], want["loss"] / 2, 1e-6 * (1 + float(want["loss"].detach())), "loss")
            assert not bool(got["dlogits"][:2].any())
        else:
            assert float(got["loss"]) == loss
        assert not bool(got["dlogits"].isnan().any())


def test_preference_far_margins_and_what_does_not_count():
    """Margins of hundreds either way (no overflow), NaN where nothing counts."""
    z, y, mask, old, ref, g = policy_inputs(6, 20, 343, BF16, 8)
    on = plain.counting(y, mask, 343)
    z = torch.where(on[..., None], z, math.nan)
    ref = torch.where(on, ref, math.nan)
    ref[0] += 30.0
    ref[2] -= 30.0
    check_preference(z, y, mask, ref, beta=2.0)
    check_preference(z, y, mask, ref, beta=2.0, smoothing=0.3)


# ---- distillation -------------------------------------------------------------------------------------------------------

def lists(z, K, g, dtype, ids_dtype, tau=1.0, spread=0.7):
    t = z.float() + spread * torch.randn(z.shape, generator=g, device=DEV)
    val, ids = torch.topk(t, K, -1)
    return val.to(dtype), ids.to(ids_dtype), torch.logsumexp(t.double() / tau, -1).float()


def check_distill(z, values, ids, **kw):
    V, tau = z.shape[2], kw.get("temperature", 1.0)
    got = ops.distill_score(z, values, ids, **kw)
    leaf, want = plain.distill(z, values, ids, **kw)
    w = kw.get("weights")
    fin = z if w is None else z[w > 0]
    tol = plain.lp_tolerance(fin if fin.numel() else z.new_zeros(1), V, tau)
    # kl = sum q (t - z) / tau + Q (lse_p - lse_q): lse_p is off by lp's error, q by a few roundings of the largest exponent
    fv = values[torch.isfinite(values)].double()
    far = float((fv.max() - fv.min()).abs() / tau) if fv.numel() else 0.0
    reach = far + float(fin[torch.isfinite(fin)].double().abs().max() / tau if fin.numel() else 0) + math.log(V) + 1
    qtol = 2.0 ** -24 * (6 + 3 * reach)
    ktol = 2 * tol + 4 * qtol * reach
    near(got["kl"], want["kl"], ktol + 2.0 ** -23 * want["kl"].abs(), "kl")
    total = tau ** 2 * (1.0 if kw.get("inv_n") is None else kw["inv_n"] * float((w if w is not None else torch.ones_like(z[..., 0])).clamp(min=0).sum()))
    near(got["loss"], want["loss"], total * ktol + 2.0 ** -22 * float(want["loss"].detach().abs()), "loss")
    check_gradient(got["dlogits"], leaf, want["loss"], z.dtype, 2 * tol + 4 * qtol, "distill")
    return got


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", FORMS + LONG)
def test_distill_vocabularies(V, dtype):
    B, T = (4, 7) if V < 20000 else (2, 3)
    z, y, mask, g = logits_of(B, T, V, dtype, V + 2, layout="sliced" if V % 2 else "plain")
    K = min(V, 24)
    val, ids, lse = lists(z, K, g, F32, torch.int32)
    w = torch.where(mask, torch.rand(B, T, generator=g, device=DEV), 0.0)
    check_distill(z, val, ids, weights=w)
    check_distill(z, val, ids, t_lse=lse, temperature=1.0)


@pytest.mark.parametrize("K", [1, 2, 15, 16, 17, 63, 64, 65, 100, 128])
@pytest.mark.parametrize("V", [343, 1367, 5463])
def test_distill_lists(K, V):
    """Every list length, both id types and value types, temperatures; ids that repeat, that are outside, entries of -inf,
    lists without an entry."""
    for k, (tau, vt, it) in enumerate([(1.0, BF16, torch.int64), (2.5, F32, torch.int32), (0.6, F32, torch.int64)]):
        z, y, mask, g = logits_of(4, 9, V, (F32, BF16)[k % 2], K + k)
        val, ids, lse = lists(z, K, g, vt, it, tau)
        if K > 2:
            ids[0, 0, 1] = ids[0, 0, 0]          # twice
            ids[0, 1, :] = ids[0, 1, 0].clone()  # all the same
            ids[0, 2, K // 2:] = -1
            ids[0, 3, 1] = V
            ids[0, 4, 0] = 2 ** 31 - 1
            val[0, 5, 1:] = -math.inf
        ids[0, 6] = -1                           # none
        val[0, 7] = -math.inf
        got = check_distill(z, val, ids, temperature=tau)
        assert float(got["kl"][0, 6]) == 0 and bool((got["dlogits"][0, 6:8] == 0).all())
        check_distill(z, val, ids, temperature=tau, t_lse=lse, inv_n=0.05)


@pytest.mark.parametrize("V", [25000, 87383, 190000])
def test_distill_long_lists_of_long_rows(V):
    """Lists of 128 of rows that a workgroup holds or walks: ids that share their low 16 bits, ids that repeat, and both."""
    for dtype in (BF16, F32):
        z, y, mask, g = logits_of(2, 3, V, dtype, V)
        val, ids, lse = lists(z, 128, g, F32, torch.int64)
        if V > 70000:
            ids[0, 0, 1] = ids[0, 0, 0] % 65536
            ids[0, 0, 2] = ids[0, 0, 0] % 65536 + 65536 if int(ids[0, 0, 0]) % 65536 + 65536 < V else ids[0, 0, 0] % 65536
        ids[0, 1, 7:9] = ids[0, 1, 100].clone()
        ids[0, 2, ::2] = ids[0, 2, 127].clone()
        ids[1, 0, 5], ids[1, 0, 6] = 2 ** 40, -2 ** 40
        check_distill(z, val, ids)
        check_distill(z, val, ids, t_lse=lse, temperature=1.0, inv_n=0.2)


def test_distill_many_tokens():
    """More tokens than one pass of the rows' kernel counts by itself: the weights summed in a launch of their own."""
    for B, T, V in ((2, 1024, 50), (1, 2049, 50), (70, 60, 343)):
        z, y, mask, g = logits_of(B, T, V, BF16, B + T)
        val, ids, lse = lists(z, 8, g, BF16, torch.int32)
        check_distill(z, val, ids, weights=torch.where(mask, torch.rand(B, T, generator=g, device=DEV), 0.0))


def test_distill_what_does_not_count():
    z, y, mask, g = logits_of(5, 8, 343, F32, 12)
    val, ids, lse = lists(z, 8, g, F32, torch.int32)
    w = torch.where(mask, 1.0, 0.0)
    w[0, 0], w[0, 1] = -1.0, math.nan
    off = ~(w > 0)
    z2, val2 = torch.where(off[..., None], math.nan, z), torch.where(off[..., None], math.nan, val)
    got = check_distill(z2, val2, ids, weights=torch.nan_to_num(w), t_lse=torch.where(off, math.nan, lse))
    again = ops.distill_score(z2, val2, ids, weights=w, t_lse=torch.where(off, math.nan, lse))
    assert torch.equal(got["dlogits"], again["dlogits"]) and bool((again["dlogits"][off] == 0).all())
    none = ops.distill_score(z2, val2, ids, weights=torch.zeros_like(w))
    assert float(none["loss"]) == 0 and bool((none["dlogits"] == 0).all()) and bool((none["kl"] == 0).all())


def test_distill_from_itself_is_zero():
    """A model against its own list: no divergence beyond the roundings of its log-sum-exp, the gradient of what the list
    leaves out alone."""
    z, y, mask, g = logits_of(3, 5, 1367, F32, 13)
    val, ids, lse = ops.top_logits(z, 128)
    got = ops.distill_score(z, val, ids, t_lse=lse)
    near(got["kl"], torch.zeros_like(got["kl"]), 4 * plain.lp_tolerance(z, 1367), "kl")


# ---- the lists ----------------------------------------------------------------------------------------------------------

def plain_top(z, k, tau):
    """By (value, lower id), from a stable sort in 64 bits; -inf and NaN are no entries."""
    x = torch.where(z > -math.inf, z.double(), -math.inf)
    val, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    val, ids = val[..., :k], ids[..., :k].clone()
    ids[val == -math.inf] = -1
    return val, ids.int(), torch.logsumexp(z.double() / tau, -1)


def check_top(z, k, tau=1.0):
    val, ids, lse = ops.top_logits(z, k, tau)
    wv, wi, wl = plain_top(z, k, tau)
    assert val.dtype == z.dtype and ids.dtype == torch.int32 and lse.dtype == F32
    assert torch.equal(val.double(), wv) and torch.equal(ids, wi)
    fin = torch.isfinite(wl)
    near(lse[fin], wl[fin], plain.lp_tolerance(z, z.shape[-1], tau) + 2.0 ** -23 * (wl[fin].abs().max() if bool(fin.any()) else 0),
         "lse")
    assert torch.equal(lse[~fin].isnan(), wl[~fin].isnan()) and bool((lse[~fin & ~wl.isnan()] == wl[~fin & ~wl.isnan()]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", FORMS + LONG)
def test_top_vocabularies(V, dtype):
    rows = (4, 5) if V < 20000 else (2, 2)
    z, y, mask, g = logits_of(*rows, V, dtype, V + 3, layout="sliced" if V % 2 else "turned")
    for k in sorted({1, min(V, 8), min(V, 33), min(V, 64), min(V, 100), min(V, 128)}):
        check_top(z, k, 1.0 if k % 2 else 2.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [7, 343, 1367, 5463, 25000, 100003, 200000])
def test_top_equal_logits(V, dtype):
    """Rows of one value, of two and three, of both zeros; negative ones; the equal ones spread or in one place."""
    g = torch.Generator(DEV).manual_seed(V)
    rows = [torch.zeros(V, device=DEV), torch.full((V,), -3.5, device=DEV),
            torch.randint(0, 2, (V,), generator=g, device=DEV).float(), torch.randint(-1, 2, (V,), generator=g, device=DEV).float(),
            torch.where(torch.rand(V, generator=g, device=DEV) < 0.5, 0.0, -0.0),
            -torch.arange(V, device=DEV).float().div(300).floor(), torch.arange(V, device=DEV).float().div(300).floor(),
            torch.where(torch.arange(V, device=DEV) == V - 1, 1.0, -1.0)]
    z = torch.stack(rows).to(dtype)
    for k in sorted({1, min(V, 64), min(V, 128)}):
        check_top(z, k)


@pytest.mark.parametrize("V", [7, 343, 5463, 87383, 200001])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_top_log_sum_exp_of_rows_with_nan(V, dtype):
    """NaN wherever a logit is, whatever the others are; the lists are of the others."""
    z = torch.zeros(6, V, dtype=dtype, device=DEV)
    z[0] = math.nan
    z[1, V // 2:] = math.nan
    z[2] = -math.inf
    z[2, V - 1] = math.nan
    z[3, 0], z[3, 3] = math.inf, math.nan
    z[4] = -math.inf
    z[5, 1] = math.inf
    values, ids, lse = ops.top_logits(z, 2)
    assert bool(lse[:4].isnan().all()) and lse[4] == -math.inf and lse[5] == math.inf
    assert ids.tolist() == [[-1, -1], [0, 1], [-1, -1], [0, 1], [-1, -1], [1, 0]]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [7, 343, 5463, 45000])
def test_top_nothing_and_infinities(V, dtype):
    """-inf, NaN and +inf among the logits, rows with fewer entries than the list or none."""
    g = torch.Generator(DEV).manual_seed(V)
    z = torch.randn(6, V, generator=g, device=DEV).to(dtype)
    z[0, torch.rand(V, generator=g, device=DEV) < 0.97] = -math.inf
    z[1] = -math.inf
    z[2] = -math.inf
    z[2, V // 2] = torch.finfo(dtype).min
    z[3, ::2] = torch.finfo(dtype).min
    z[4, 3] = math.nan
    z[5, 2], z[5, 5] = math.inf, math.inf
    for k in sorted({1, min(V, 5), min(V, 128)}):
        val, ids, lse = ops.top_logits(z, k)
        wv, wi, wl = plain_top(z, k, 1.0)
        assert torch.equal(val.double(), wv) and torch.equal(ids, wi)
        assert float(lse[1]) == -math.inf and bool(lse[4].isnan())
        near(lse[[0, 2, 3]], wl[[0, 2, 3]], 2.0 ** -22 * wl[[0, 2, 3]].abs() + 2e-5, "lse")


def test_top_many_rows():
    for rows, V, k in ((5000, 7, 3), (9000, 343, 32), (3000, 1367, 64), (2500, 5463, 16)):
        g = torch.Generator(DEV).manual_seed(rows)
        check_top(torch.randn(rows, V, generator=g, device=DEV).to(BF16), k)


# ---- the differentiable forms -------------------------------------------------------------------------------------------

def objective_calls(dtype=BF16, V=343, seed=21):
    z, y, mask, old, ref, g = policy_inputs(4, 12, V, dtype, seed, far=0.05)
    val, ids, lse = lists(z, 9, g, F32, torch.int32)
    adv = torch.randn(4, generator=g, device=DEV)
    return z, [
        (objectives.token_policy_loss, ops.policy_score, plain.policy,
         dict(targets=y, mask=mask, old_lp=old, adv=adv, ref_lp=ref, kl_coef=0.1)),
        (objectives.preference_loss, ops.preference_score, plain.preference, dict(targets=y, mask=mask, ref_lp=ref)),
        (objectives.distill_loss, ops.distill_score, plain.distill, dict(values=val, ids=ids, t_lse=lse)),
    ]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_backward_hands_out_what_score_computes(which):
    z, calls = objective_calls()
    loss_fn, score, _, kw = calls[which]
    leaf = z.clone().requires_grad_(True)
    want = score(z, **kw)
    out = loss_fn(leaf, **kw)
    assert torch.equal(out[0], want["loss"]) and out[0].requires_grad
    assert not any(t.requires_grad for t in out[1:] if t is not None)
    out[0].backward(retain_graph=True)
    assert torch.equal(leaf.grad, want["dlogits"])
    first = leaf.grad
    again = torch.autograd.grad(out[0], leaf, retain_graph=True)[0]   # anew: the first one is the leaf's own now
    assert torch.equal(again, want["dlogits"]) and again.data_ptr() != first.data_ptr()
    # a factor of the loss: rounded once
    for factor in (0.37, -2.0, 0.0, 1.0):
        got = torch.autograd.grad(factor * loss_fn(leaf, **kw)[0], leaf)[0]
        up = torch.tensor(factor, device=DEV)
        assert torch.equal(got, score(z, **kw, upstream=up)["dlogits"])
        f = score(z.float(), **kw)["dlogits"].double() * float(up)
        near(got, f, torch.finfo(BF16).eps / 2 * f.abs() * (1 + 1e-4) + 1e-9 * f.abs().max() + 1e-37, "factor")
    with torch.no_grad():  # no gradient, nor its memory
        before = torch.cuda.memory_allocated()
        off = loss_fn(leaf, **kw)
        assert not off[0].requires_grad and torch.cuda.memory_allocated() - before < leaf.numel()
        assert torch.equal(off[0], want["loss"])
    leaf.grad = None
    (loss_fn(leaf, **kw)[0] + loss_fn(leaf, **kw)[0]).backward()
    near(leaf.grad, 2 * want["dlogits"].double(), torch.finfo(BF16).eps * want["dlogits"].double().abs() + 1e-37, "sum of two")


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("layout", ["plain", "sliced"])
def test_backward_of_moved_tensors(which, layout):
    """Saved tensors that hooks move to the host and back (contiguous then), and a checkpointed region that is computed
    anew: the gradient of a scaled loss, and of a kept graph's second backward, reads what the hooks give."""
    z, calls = objective_calls()
    if layout == "sliced":
        big = torch.zeros(4, 15, 348, dtype=BF16, device=DEV)
        big[:, 2:14, 3:346] = z
        z = big[:, 2:14, 3:346]
    loss_fn, score, _, kw = calls[which]
    want = score(z, **kw, upstream=torch.tensor(0.37, device=DEV))["dlogits"]
    leaf = z.detach().requires_grad_(True)
    with torch.autograd.graph.save_on_cpu():
        loss = loss_fn(leaf * 1, **kw)[0]
        view = loss_fn(leaf, **kw)[0]
    torch.empty(4, 12, 343, dtype=BF16, device=DEV).fill_(math.nan)  # (memory that the product's result may have had)
    assert torch.equal(torch.autograd.grad(0.37 * loss, leaf, retain_graph=True)[0], want)
    assert torch.equal(torch.autograd.grad(0.37 * loss, leaf)[0], want)
    assert torch.equal(torch.autograd.grad(0.37 * view, leaf)[0], want)
    again = torch.utils.checkpoint.checkpoint(lambda x: loss_fn(x * 1, **kw)[0], leaf, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(0.37 * again, leaf)[0], want)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_backward_of_logits_laid_out_anew_at_their_address(which):
    """Hooks that give the logits back at the address they had, their rows packed: the strides are the packed ones. Kept
    inputs of another type or size, or on the host, are refused."""
    z, calls = objective_calls()
    loss_fn, score, _, kw = calls[which]
    want = score(z, **kw, upstream=torch.tensor(0.37, device=DEV))["dlogits"]
    big = torch.zeros(4, 15, 348, dtype=BF16, device=DEV)
    view = big[:, 2:14, 3:346]
    view.copy_(z)
    leaf = view.detach().requires_grad_(True)

    def pack(t):
        return t.clone(memory_format=torch.contiguous_format)

    def unpack(t):
        if t.shape != z.shape or t.dtype is not BF16:
            return t
        big.zero_()
        there = big.view(-1)[view.storage_offset():][:t.numel()].view(t.shape)
        assert there.data_ptr() == view.data_ptr()
        return there.copy_(t)

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        loss = loss_fn(leaf, **kw)[0]
    assert torch.equal(torch.autograd.grad(0.37 * loss, leaf, retain_graph=True)[0], want)
    assert torch.equal(torch.autograd.grad(0.37 * loss, leaf)[0], want)

    def halves(t):
        return t.bfloat16() if t.dtype is torch.float32 else t[:2] if t.dtype is torch.uint8 else t

    for give in (halves, lambda t: t[:, :-1] if t.shape == z.shape else t, lambda t: t.cpu() if t.dim() == 2 else t,
                 lambda t: t.cpu()):
        leaf = z.detach().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, give):
            loss = loss_fn(leaf, **kw)[0]
        with pytest.raises(AssertionError, match="kept"):
            loss.backward()


def test_inputs_written_to_before_the_backward():
    """Autograd's own refusal: an input of the loss that changed in between."""
    z, calls = objective_calls()
    for loss_fn, _, _, kw in calls:
        leaf = z.clone().requires_grad_(True)
        x = leaf * 1
        loss = loss_fn(x, **kw)[0]
        x.data.add_(0)  # (no version: still good)
        loss.backward(retain_graph=True)
        with torch.no_grad():
            x.add_(1)
        with pytest.raises(RuntimeError):
            loss.backward()


@pytest.mark.parametrize("which", [0, 1, 2])
def test_gradient_against_differences(which):
    """Central differences of the 64-bit definition along random directions. Its third derivative along a direction of
    length 1 is at most a few units, so that steps of 1e-4 leave 1e-8, and the 64-bit losses 1e-12 / 1e-4; the kernel's
    gradient in fp32 is off by 1e-6 of its length."""
    z, calls = objective_calls(F32, 33, 5)
    _, score, definition, kw = calls[which]
    got = score(z, **kw)["dlogits"].double()
    g = torch.Generator(DEV).manual_seed(1)
    for _ in range(8):
        d = torch.randn(z.shape, generator=g, device=DEV, dtype=torch.float64)
        d /= d.norm()
        h = 1e-4
        up, down = (float(definition(z.double() + s * h * d, **kw)[1]["loss"].detach()) for s in (1, -1))
        assert abs((up - down) / (2 * h) - float((got * d).sum())) < 2e-7 + 2e-5 * float(got.norm())


def test_same_bits_every_run():
    z, calls = objective_calls(BF16, 5463)
    for _, score, _, kw in calls:
        a = score(z, **kw)
        for _ in range(3):
            b = score(z, **kw)
            assert all(torch.equal(a[k], b[k]) for k in a if a[k] is not None)


def test_forms_agree():
    """The same tokens alone and in a batch: rows do not depend on what is beside them."""
    z, y, mask, old, ref, g = policy_inputs(40, 30, 1367, BF16, 2)
    mask[:] = True
    adv = torch.randn(40, generator=g, device=DEV)
    all_ = ops.policy_score(z, y, mask, old, adv, ref, kl_coef=0.1, per="token", inv_n=1.0)
    one = ops.policy_score(z[7:8], y[7:8], mask[7:8], old[7:8], adv[7:8], ref[7:8], kl_coef=0.1, per="token", inv_n=1.0)
    assert torch.equal(all_["dlogits"][7:8], one["dlogits"]) and torch.equal(all_["lp"][7:8], one["lp"])


def test_empty_calls():
    for B, T in ((0, 5), (3, 0), (0, 0)):
        z = torch.empty(B, T, 343, device=DEV)
        y, m = torch.empty(B, T, dtype=torch.long, device=DEV), torch.empty(B, T, dtype=torch.bool, device=DEV)
        f = torch.empty(B, T, device=DEV)
        r = ops.policy_score(z, y, m, f, torch.empty(B, device=DEV), f)
        assert float(r["loss"]) == 0 and r["dlogits"].shape == z.shape
        if B % 2 == 0:
            r = ops.preference_score(z, y, m, f)
            assert float(r["loss"]) == 0 and r["margin"].shape == (B // 2,)
        r = ops.preference_score(z, y, m, f, pairs=torch.zeros(2, 2, dtype=torch.long, device=DEV))
        assert math.isfinite(float(r["loss"])) and r["margin"].tolist() == [0.0, 0.0]
        r = ops.distill_score(z, torch.empty(B, T, 4, device=DEV), torch.empty(B, T, 4, dtype=torch.int32, device=DEV))
        assert float(r["loss"]) == 0 and r["kl"].shape == (B, T)
        val, ids, lse = ops.top_logits(z, 4)
        assert val.shape == (B, T, 4) and lse.shape == (B, T)


def test_past_32_bit_offsets():
    """2^31 + elements of logits: the last rows' results."""
    B, T, V = 5, 5000, 87383
    z = torch.zeros(B, T, V, dtype=BF16, device=DEV)
    assert z.numel() > 2 ** 31
    g = torch.Generator(DEV).manual_seed(9)
    tail, y1, _, _ = logits_of(1, 3, V, BF16, 9)
    z[-1:, -3:] = tail
    y = torch.zeros(B, T, dtype=torch.long, device=DEV)
    y[-1:, -3:] = y1
    mask = torch.zeros(B, T, dtype=torch.bool, device=DEV)
    mask[-1, -3:] = True
    old = torch.full((B, T), -1.0, device=DEV)
    got = ops.policy_score(z, y, mask, old, torch.ones(B, device=DEV), per="token")
    one = ops.policy_score(z[-1:, -3:], y1, mask[-1:, -3:], old[-1:, -3:], torch.ones(1, device=DEV), per="token")
    assert torch.equal(got["dlogits"][-1:, -3:], one["dlogits"]) and float(got["dlogits"][0].abs().max()) == 0
    got = ops.preference_score(z, y, mask, old, pairs=torch.tensor([[B - 1, 0]], device=DEV), out=got["dlogits"])
    one = ops.preference_score(z[-1:, -3:], y1, mask[-1:, -3:], old[-1:, -3:], pairs=torch.tensor([[0, 0]], device=DEV))
    assert torch.equal(got["lp"][-1:, -3:], one["lp"]) and float(got["dlogits"][-1, -1].float().abs().max()) > 0
    val, ids, lse = ops.top_logits(z, 16)
    v1, i1, l1 = ops.top_logits(z[-1:, -3:], 16)
    assert torch.equal(ids[-1:, -3:], i1) and torch.equal(val[-1:, -3:], v1) and torch.equal(lse[-1:, -3:], l1)
    w = mask.float()
    got = ops.distill_score(z, val.float() + 0.3 * torch.rand(B, T, 16, device=DEV), ids, weights=w, out=got["dlogits"])
    assert float(got["dlogits"][0].abs().max()) == 0 and float(got["dlogits"][-1, -1].float().abs().max()) > 0


# ---- streams and graphs -------------------------------------------------------------------------------------------------

def test_side_stream():
    z, calls = objective_calls()
    wants = [score(z, **kw) for _, score, _, kw in calls]
    top = ops.top_logits(z, 20)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        gots = [score(z, **kw) for _, score, _, kw in calls]
        top2 = ops.top_logits(z, 20)
    side.synchronize()
    for a, b in zip(wants, gots):
        assert all(torch.equal(a[k], b[k]) for k in a if a[k] is not None)
    assert all(torch.equal(a, b) for a, b in zip(top, top2))


def test_two_streams_at_once():
    """Calls of different inputs on two streams, nothing between them: each as alone."""
    sets = [objective_calls(BF16, 5463, seed) for seed in (1, 2)]
    wants = [[score(z, **kw) for _, score, _, kw in calls] for z, calls in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    gots = [[], []]
    for _ in range(3):
        for i, (z, calls) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                gots[i] += [score(z, **kw) for _, score, _, kw in calls]
    torch.cuda.synchronize()
    for want, got in zip(wants, gots):
        for k, b in enumerate(got):
            a = want[k % 3]
            assert all(torch.equal(a[n], b[n]) for n in a if a[n] is not None)


def test_captured_and_replayed():
    """Scores, and losses with their backward, in one captured graph, replayed on new inputs with eager work between."""
    z, calls = objective_calls()
    leaf = z.clone().requires_grad_(True)

    def program():
        outs = []
        for loss_fn, score, _, kw in calls:
            outs += [v for k, v in score(leaf.detach(), **kw).items() if v is not None]
            loss = loss_fn(leaf, **kw)[0]
            outs += [loss.detach(), *torch.autograd.grad(loss * 0.5, leaf)]
            outs += torch.autograd.grad(loss_fn(leaf, **kw)[0], leaf)
        outs += ops.top_logits(leaf.detach(), 12)
        return [o.detach() for o in outs]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(2):
            program()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = program()
    for k in range(4):
        with torch.no_grad():
            leaf.copy_(logits_of(4, 12, 343, BF16, 100 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in kept]
        want = program()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


@pytest.mark.parametrize("which", [0, 1, 2])
def test_backward_captured_without_its_forward_computes_the_gradient(which, monkeypatch):
    """Its replays would find what the last user of the gradient left in it: it is not taken from the forward then."""
    z, calls = objective_calls()
    loss_fn, score, _, kw = calls[which]
    want = score(z, **kw)["dlogits"]
    leaf = z.clone().requires_grad_(True)
    for captured in (True, False):
        monkeypatch.setattr(objectives, "_capturing", lambda: False)
        loss = loss_fn(leaf, **kw)[0]
        loss.grad_fn.dlogits.zero_()
        monkeypatch.setattr(objectives, "_capturing", lambda: captured)
        got = torch.autograd.grad(loss, leaf)[0]
        assert torch.equal(got, want if captured else torch.zeros_like(want))


# ---- refusals that need device tensors ----------------------------------------------------------------------------------

def test_refusals():
    z, y, mask, old, ref, g = policy_inputs(4, 6, 33, F32, 1)
    adv = torch.ones(4, device=DEV)
    val, ids, lse = ops.top_logits(z, 5)
    bad_policy = [dict(logits=z[0]), dict(logits=z.half()), dict(logits=z.expand(4, 6, 33)[:, :1].expand(4, 6, 33)),
                  dict(logits=z.transpose(1, 2)), dict(targets=y.int()), dict(targets=y[:, 1:]), dict(mask=mask.float()),
                  dict(mask=mask[:1]), dict(old_lp=old.double()), dict(old_lp=old[:1]), dict(old_lp=None), dict(adv=adv[:2]),
                  dict(adv=adv.double()), dict(ref_lp=ref[:, :2]), dict(kl_coef=0.1, ref_lp=None), dict(per="batch"),
                  dict(eps_lo=-0.1), dict(out=torch.empty(4, 6, 33, device=DEV, dtype=BF16)), dict(out=z), dict(out=z[:, :3]),
                  dict(upstream=adv), dict(out=torch.empty_like(z), grad=False),
                  dict(targets=y.cpu()), dict(upstream=torch.ones((), dtype=torch.float64, device=DEV))]
    for kw in bad_policy:
        with pytest.raises((AssertionError, RuntimeError)):
            ops.policy_score(**{**dict(logits=z, targets=y, mask=mask, old_lp=old, adv=adv, ref_lp=ref), **kw})
    for kw in (dict(logits=z[:3], targets=y[:3], mask=mask[:3], ref_lp=ref[:3]), dict(pairs=torch.zeros(2, 2, device=DEV)),
               dict(pairs=torch.zeros(4, dtype=torch.long, device=DEV)), dict(lengths=adv[:1]), dict(smoothing=1.5),
               dict(smoothing=math.nan), dict(ref_lp=ref.double())):
        with pytest.raises(AssertionError):
            ops.preference_score(**{**dict(logits=z, targets=y, mask=mask, ref_lp=ref), **kw})
    for kw in (dict(values=val[..., :3]), dict(values=val.double()), dict(ids=ids.short()), dict(values=val[0], ids=ids[0]),
               dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
               dict(t_lse=lse.double()), dict(weights=lse[:1]), dict(values=val[..., :0], ids=ids[..., :0]),
               dict(values=torch.zeros(4, 6, 129, device=DEV), ids=torch.zeros(4, 6, 129, dtype=torch.int32, device=DEV))):
        with pytest.raises(AssertionError):
            ops.distill_score(**{**dict(logits=z, values=val, ids=ids), **kw})
    for args in ((z, 0), (z, 34), (torch.zeros(2, 300, device=DEV), 129), (z, 4, 0.0), (z, 4, math.inf), (z[0, 0], 3),
                 (z.double(), 3), (z.transpose(1, 2), 3)):
        with pytest.raises(AssertionError):
            ops.top_logits(*args)
