"""What the large-vocabulary entry points refuse before any launch, and their host-side helpers (no GPU)."""

import ctypes

import pytest
import torch

from viktor_amd import _lib, hip_ops as ops


def _p():
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    return ctypes.c_void_p(at), buf


def _err(rc, word):
    assert rc == 1 and word in _lib.load().vk_last_error(), (rc, _lib.load().vk_last_error())


def test_embedding_entry_points_refuse():
    lib = _lib.load()
    p, _ = _p()
    _err(lib.vk_embed_lookup(p, 0, p, 4, 0, 8, 1.0, p, 0, None), b"sizes")
    _err(lib.vk_embed_lookup(p, 0, p, 4, 9, 2 ** 20 + 1, 1.0, p, 0, None), b"sizes")
    _err(lib.vk_embed_lookup(None, 0, p, 4, 9, 8, 1.0, p, 0, None), b"null")
    _err(lib.vk_embed_lookup(p, 2, p, 4, 9, 8, 1.0, p, 0, None), b"dtype")
    need = ctypes.c_int64(0)
    _err(lib.vk_embed_grad_sorted_workspace(2 ** 31, 9, 8, ctypes.byref(need)), b"rows")
    _err(lib.vk_embed_grad_sorted_workspace(4, 9, 2 ** 20 + 1, ctypes.byref(need)), b"arguments")
    assert lib.vk_embed_grad_sorted_workspace(10000, 5463, 64, ctypes.byref(need)) == 0
    _err(lib.vk_embed_grad_sorted(p, 1, 64, p, 10000, 5463, 64, 1.0, -1, p, 0, p, need.value - 1, None), b"workspace")
    _err(lib.vk_embed_grad_sorted(p, 1, 63, p, 10000, 5463, 64, 1.0, -1, p, 0, p, need.value, None), b"sizes")
    _err(lib.vk_embed_grad_sorted(p, 7, 64, p, 10000, 5463, 64, 1.0, -1, p, 0, p, need.value, None), b"dtype")
    _err(lib.vk_embed_grad_sorted(None, 1, 64, p, 10000, 5463, 64, 1.0, -1, p, 0, p, need.value, None), b"null")


def test_embedding_workspace_covers_what_the_passes_write():
    """Grows with each size; both sorts on their sides of the border."""
    lib = _lib.load()

    def need(n, V, d):
        b = ctypes.c_int64(0)
        assert lib.vk_embed_grad_sorted_workspace(n, V, d, ctypes.byref(b)) == 0
        return b.value

    assert need(0, 7, 1) >= 16
    for n in (1, 31, 32, 64, 65, 4096, 4097, 16384, 16385, 102400, 102401, 131072, 131073, 524288, 600000):
        chunk = 16 if n <= 16384 else 32 if n <= 102400 else 64
        partials = 8 * -(-n // chunk) if n >= 2 * chunk else 0  # fp32 rows: two slots a chunk
        for V in (1, 343, 87383, 300000):
            for d in (1, 512):
                # sorted pairs of 8 bytes (two buffers past the counting sort), partial sums, the list of long runs
                assert need(n, V, d) >= (8 if n <= 4096 else 16) * n + partials * d + 4 * (-(-n // chunk) + 1)


def _process(lib, p, **kw):
    a = dict(logits=p, dtype=1, ld=40, hist=p, hist_ld=5, hist_cols=5, hist_len=p, rep=None, rep0=1.1, pres=None, pres0=0.0,
             freq=None, freq0=0.0, bias=None, bias_ld=0, allowed=None, allowed_ld=0, n_allowed=0, rows=None, out=p, odt=1,
             out_ld=40, B=3, V=40, stream=None)
    a.update(kw)
    return lib.vk_process_logits(*a.values())


def test_process_logits_refuses():
    lib = _lib.load()
    p, _ = _p()
    q = ctypes.c_void_p(p.value + 64)
    for kw, word in (({"ld": 39}, b"sizes"), ({"V": 0}, b"sizes"), ({"dtype": 3}, b"bf16 or fp32"), ({"logits": None}, b"null"),
                     ({"odt": 9}, b"out"), ({"out_ld": 39}, b"out"), ({"odt": 0}, b"in place"), ({"out_ld": 48}, b"in place"),
                     ({"hist_len": None}, b"lengths"), ({"hist_cols": 65536, "hist_ld": 65536}, b"65535"), ({"hist_ld": 4}, b"65535"),
                     ({"rep0": 0.0}, b"positive"), ({"rep0": float("nan")}, b"positive"), ({"bias": q, "bias_ld": 7}, b"bias"),
                     ({"allowed": q, "allowed_ld": 1, "n_allowed": 1}, b"words"), ({"allowed": q, "allowed_ld": 2, "n_allowed": 0}, b"words"),
                     ({"allowed": q, "allowed_ld": 2, "n_allowed": 2}, b"row numbers"), ({"B": 2 ** 20}, b"sequences"), ({"V": 2 ** 30 + 1, "ld": 2 ** 31}, b"sizes"),
                     ({"B": 2 ** 19, "V": 2 ** 20, "ld": 2 ** 20, "out_ld": 2 ** 20}, b"too many")):
        _err(_process(lib, p, **kw), word)
    assert _process(lib, p, B=0) == 0


def _choose(lib, p, **kw):
    a = dict(logits=p, dtype=1, ld=40, hist=None, hist_ld=0, hist_cols=0, hist_len=None, rep=None, rep0=1.0, pres=None, pres0=0.0,
             freq=None, freq0=0.0, bias=None, bias_ld=0, allowed=None, allowed_ld=0, n_allowed=0, rows=None, temp=None, temp0=0.0,
             mode=0, uniforms=None, u_ld=0, fallback=0, token=p, logp=None, B=3, V=40, ws=p, ws_bytes=4096, stream=None)
    a.update(kw)
    return lib.vk_choose_tokens(*a.values())


def test_choose_tokens_refuses():
    lib = _lib.load()
    p, _ = _p()
    big = {"V": 87383, "ld": 87383}  # (needs a workspace)
    for kw, word in (({"token": None}, b"null"), ({"mode": 3}, b"mode"), ({"mode": 1}, b"uniforms"),
                     ({"mode": 1, "uniforms": p, "u_ld": 39}, b"uniforms"), ({"mode": 2, "uniforms": p, "u_ld": 0}, b"uniforms"),
                     ({"B": 2 ** 19, "V": 2 ** 20, "ld": 2 ** 20}, b"too many"), ({"V": 2 ** 30 + 1, "ld": 2 ** 31}, b"sizes"),
                     ({**big, "ws": None}, b"workspace"), ({**big, "ws_bytes": 16}, b"workspace"),
                     ({**big, "ws": ctypes.c_void_p(p.value + 4)}, b"workspace")):
        _err(_choose(lib, p, **kw), word)
    assert _choose(lib, p, B=0) == 0
    need = ctypes.c_int64(0)
    assert lib.vk_choose_tokens_workspace(0, 40, 0, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.vk_choose_tokens_workspace(3, 40, 5, ctypes.byref(need)) == 0 and need.value == 0  # one launch
    assert lib.vk_choose_tokens_workspace(3, 87383, 5, ctypes.byref(need)) == 0 and need.value > 0
    _err(lib.vk_choose_tokens_workspace(-1, 40, 0, ctypes.byref(need)), b"arguments")
    _err(lib.vk_choose_tokens_workspace(1, 2 ** 31 - 1, 0, ctypes.byref(need)), b"arguments")


def test_choose_update_refuses():
    lib = _lib.load()
    p, _ = _p()

    def step(**kw):
        a = dict(logits=p, dtype=1, ld=40, rep0=1.0, pres0=0.0, freq0=0.0, bias=p, allowed=None, allowed_ld=0, n_allowed=0,
                 token_rows=None, is_tail=p, is_homo=p, homo_stop=0, temperature=0.0, mode=0, uniforms=None, u_ld=0, u_cols=0,
                 tok=p, run=p, pos=p, plen=None, rope_off=None, cache_base=None, out=p, out_stride=8, out_cols=8, pos32=None,
                 seqlens=None, rpos32=None, logp=None, logp_stride=0, B=3, V=40, eos=2, pad=0, ws=p, ws_bytes=4096, stream=None)
        a.update(kw)
        return lib.vk_choose_update(*a.values())

    for kw, word in (({"tok": None}, b"null"), ({"bias": None}, b"null"), ({"homo_stop": 4, "run": None}, b"run"),
                     ({"out_stride": 7}, b"rows"), ({"out_cols": 0}, b"rows"), ({"logp": p, "logp_stride": 7}, b"logp_stride"),
                     ({"allowed": p, "allowed_ld": 2, "n_allowed": 1}, b"mask row"), ({"rep0": -1.0}, b"positive"),
                     ({"mode": 1, "uniforms": p, "u_cols": 8, "u_ld": 8 * 40 - 1}, b"uniforms"),
                     ({"mode": 2, "uniforms": p, "u_cols": 8, "u_ld": 7}, b"uniforms"), ({"rep0": 1.1, "out_cols": 70000, "out_stride": 70000}, b"65535")):
        _err(step(**kw), word)
    assert step(B=0) == 0


def test_wrappers_refuse_cpu_tensors():
    z, tok = torch.zeros(3, 40), torch.zeros(6, dtype=torch.long)
    for f in (lambda: ops.embed_lookup(torch.zeros(40, 8), tok), lambda: ops.embed_grad_sorted(torch.zeros(6, 8), tok, 40),
              lambda: ops.process_logits(z), lambda: ops.choose_tokens(z)):
        with pytest.raises(_lib.HipLibraryError):
            f()


def test_pack_allowed():
    for V in (1, 31, 32, 33, 343, 1367):
        mask = torch.rand(4, V, generator=torch.Generator().manual_seed(V)) < 0.5
        mask[0] = True
        words = ops.pack_allowed(mask)
        assert words.shape == (4, -(-V // 32)) and words.dtype == torch.int32
        v = torch.arange(V)
        assert torch.equal(((words.long()[:, v // 32] >> (v % 32)) & 1).bool(), mask)
        if V % 32:
            assert not bool((words[0, -1].long() & 0xffffffff) >> (V % 32))
    with pytest.raises(AssertionError):
        ops.pack_allowed(torch.zeros(4, 8))
