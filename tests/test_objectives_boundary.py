"""What the entry points of the objectives on logits refuse before any launch (no GPU)."""

import ctypes

import pytest
import torch

from viktor_amd import _lib, hip_ops as ops, objectives


def _p():
    buf = ctypes.create_string_buffer(1 << 17)
    return ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16), buf


def _err(rc, word):
    assert rc == 1 and word in _lib.load().vk_last_error(), (rc, _lib.load().vk_last_error())


def _workspace(B, T, P):
    n = ctypes.c_int64(0)
    assert _lib.load().vk_objective_workspace(B, T, P, ctypes.byref(n)) == 0
    return n.value


def test_workspace_covers_what_the_passes_write():
    lib = _lib.load()
    n = ctypes.c_int64(0)
    _err(lib.vk_objective_workspace(1, 1, 0, None), b"arguments")
    _err(lib.vk_objective_workspace(-1, 1, 0, ctypes.byref(n)), b"arguments")
    _err(lib.vk_objective_workspace(2 ** 16, 2 ** 15, 0, ctypes.byref(n)), b"arguments")
    _err(lib.vk_objective_workspace(1, 1, 2 ** 31, ctypes.byref(n)), b"arguments")
    for B, T in ((0, 0), (1, 1), (512, 1024), (3, 100000)):
        # partial sums of 64 bits, a 32-bit count per sequence
        assert _workspace(B, T, 0) >= 8 * (256 + 2048) + 4 * B
        for P in (1, 7, 1000):
            # per sequence a 64-bit ratio and a 32-bit slope, per pair a 64-bit slope, per token 12 bytes
            assert _workspace(B, T, P) >= 12 * B + 8 * P + 12 * B * T


SIZES = [({"dtype": 2}, b"bf16 or fp32"), ({"V": 0}, b"sizes"), ({"V": 2 ** 30 + 1, "ld_t": 2 ** 31, "ld_b": 2 ** 33}, b"sizes"),
         ({"B": -1}, b"sizes"), ({"T": 2 ** 31}, b"sizes"), ({"B": 2 ** 16, "T": 2 ** 15}, b"sizes"), ({"logits": None}, b"null"),
         ({"ld_t": 39}, b"overlap"), ({"ld_b": 39}, b"overlap"), ({"ws": None}, b"workspace"), ({"ws_bytes": 64}, b"workspace")]


def _policy(p, **kw):
    a = dict(logits=p, dtype=1, ld_b=200, ld_t=40, targets=p, mask=p, old=p, adv=p, adv2=0, ref=p, lo=0.2, hi=0.2, coef=0.1, per=0,
             inv=1.0, loss=p, pg=p, kl=p, lp=p, d=p, up=None, unless=0, B=3, T=5, V=40, ws=p, ws_bytes=1 << 16, stream=None)
    a.update(kw)
    return _lib.load().vk_policy_score(*a.values())


def test_policy_refuses():
    p, _ = _p()
    for kw, word in SIZES + [({"per": 3}, b"per"), ({"ref": None}, b"ref_lp"), ({"ref": None, "coef": 0.0}, b"kl needs"),
                             ({"unless": 1}, b"upstream"), ({"targets": None}, b"null"), ({"mask": None}, b"null"),
                             ({"old": None}, b"null"), ({"adv": None}, b"null"),
                             ({"ws": ctypes.c_void_p(p.value + 8)}, b"workspace")]:
        _err(_policy(p, **kw), word)


def _preference(p, **kw):
    a = dict(logits=p, dtype=1, ld_b=200, ld_t=40, targets=p, mask=p, ref=p, lengths=None, pairs=None, P=2, beta=0.1, target=0.0,
             smoothing=0.0, inv=0.5, loss=p, margin=p, lp=p, d=p, up=None, unless=0, parts=3, B=4, T=5, V=40, ws=p,
             ws_bytes=1 << 16, stream=None)
    a.update(kw)
    return _lib.load().vk_preference_score(*a.values())


def test_preference_refuses():
    p, _ = _p()
    for kw, word in SIZES + [({"P": 3}, b"pair"), ({"P": -1, "pairs": p}, b"pair"), ({"parts": 0}, b"parts"), ({"parts": 4}, b"parts"),
                             ({"unless": 1}, b"upstream"), ({"targets": None}, b"null"), ({"loss": None}, b"null output"),
                             ({"margin": None}, b"null output"), ({"lp": None}, b"null output"), ({"d": None}, b"null gradient")]:
        _err(_preference(p, **{**({"P": 2 ** 15 * 2 ** 15} if kw.get("B") == 2 ** 16 else {}), **kw}), word)


def _distill(p, **kw):
    a = dict(logits=p, dtype=1, ld_b=200, ld_t=40, values=p, vdt=1, ids=p, ids64=0, K=4, t_lse=None, weights=None, tau=1.0, mean=1,
             inv=1.0, loss=p, kl=p, d=p, up=None, unless=0, B=3, T=5, V=40, ws=p, ws_bytes=1 << 16, stream=None)
    a.update(kw)
    return _lib.load().vk_distill_score(*a.values())


def test_distill_refuses():
    p, _ = _p()
    for kw, word in SIZES + [({"K": 0}, b"lists"), ({"K": 129}, b"lists"), ({"vdt": 2}, b"list values"), ({"tau": 0.0}, b"temperature"),
                             ({"tau": float("nan")}, b"temperature"), ({"tau": float("inf")}, b"temperature"),
                             ({"unless": 1}, b"upstream"), ({"values": None}, b"null"), ({"ids": None}, b"null")]:
        _err(_distill(p, **kw), word)


def test_top_refuses():
    lib = _lib.load()
    p, _ = _p()
    for kw, word in (({"dtype": 5}, b"bf16 or fp32"), ({"V": 0}, b"sizes"), ({"B": 2 ** 31}, b"sizes"), ({"K": 0}, b"lists"),
                     ({"K": 41}, b"lists"), ({"V": 300, "ld_t": 300, "ld_b": 3000, "K": 129}, b"lists"), ({"tau": -1.0}, b"temperature"),
                     ({"logits": None}, b"null"), ({"values": None}, b"null"), ({"ids": None}, b"null"), ({"lse": None}, b"null"),
                     ({"ld_t": 39}, b"overlap"), ({"ld_b": -1}, b"overlap")):
        a = dict(logits=p, dtype=1, ld_b=200, ld_t=40, K=4, tau=1.0, values=p, ids=p, lse=p, B=3, T=5, V=40, stream=None)
        a.update(kw)
        _err(lib.vk_top_logits(*a.values()), word)
    assert lib.vk_top_logits(None, 1, 0, 0, 4, 1.0, None, None, None, 0, 5, 40, None) == 0


def test_host_tensors_are_refused():
    z, y = torch.zeros(2, 3, 7), torch.zeros(2, 3, dtype=torch.long)
    m, f = torch.ones(2, 3, dtype=torch.bool), torch.zeros(2, 3)
    lists = torch.zeros(2, 3, 2), torch.zeros(2, 3, 2, dtype=torch.int32)
    for call in (lambda: ops.policy_score(z, y, m, f, f), lambda: ops.preference_score(z, y, m), lambda: ops.distill_score(z, *lists),
                 lambda: ops.top_logits(z, 2), lambda: objectives.token_policy_loss(z, y, m, f, f),
                 lambda: objectives.preference_loss(z, y, m), lambda: objectives.distill_loss(z, *lists)):
        with pytest.raises(_lib.HipLibraryError):
            call()
