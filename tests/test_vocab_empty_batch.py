"""Empty batches of the rules on logits and the token choice: answered like a batch of rows, with every option, whatever the
pointers of the tensors without elements are."""

import ctypes

import pytest
import torch

from viktor_amd import _lib, hip_ops as ops

DEV = "cuda"


def _p():
    buf = ctypes.create_string_buffer(4096)
    return ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16), buf


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_entry_points_take_null_rows_of_an_empty_batch(mode):
    lib = _lib.load()
    p, _keep = _p()
    V = 40
    rules = [None, 5, 5, None, None, 1.1, None, 0.1, None, 0.1, p, 0]  # history of no rows .. bias
    for masks in ([None, 0, 0, None], [p, 2, 3, None], [p, 2, 1, None]):
        assert lib.vk_choose_tokens(None, 1, V, *rules, *masks, None, 0.9, mode, None, V, 0, None, None, 0, V, None, 0, None) == 0
        assert lib.vk_process_logits(None, 1, V, *rules, *masks, None, 1, V, 0, V, None) == 0
    for masks in ([None, 0, 0, None], [p, 2, 3, p]):
        assert lib.vk_choose_update(None, 1, V, 1.1, 0.0, 0.0, p, *masks, p, p, 4, 0.9, mode, None, 8 * V, 8, None, None, None,
                                    None, None, None, None, 8, 8, None, None, None, None, 0, 0, V, 2, 0, None, 0, None) == 0
    # what a batch of any size would be refused for still is
    assert lib.vk_choose_update(None, 1, V, 1.1, 0.0, 0.0, None, None, 0, 0, None, p, p, 4, 0.9, mode, None, 8 * V, 8, None, None,
                                None, None, None, None, None, 8, 8, None, None, None, None, 0, 0, V, 2, 0, None, 0, None) == 1
    if mode != 0:
        assert lib.vk_choose_tokens(None, 1, V, *rules, None, 0, 0, None, None, 0.9, mode, None, 0, 0, None, None, 0, V, None, 0,
                                    None) == 1


@pytest.mark.gpu
def test_wrappers_answer_an_empty_batch():
    V, T = 5463, 9
    z = torch.zeros(0, V, device=DEV)
    vec = lambda dt: torch.zeros(0, dtype=dt, device=DEV)  # noqa: E731
    rules = dict(history=torch.zeros(0, T, dtype=torch.long, device=DEV), lengths=vec(torch.int32), repetition=vec(torch.float32),
                 presence=0.5, frequency=vec(torch.float32), bias=torch.zeros(V, device=DEV))
    words = torch.full((3, -(-V // 32)), -1, dtype=torch.int32, device=DEV)
    for masks in ({}, {"allowed": words[:1]}, {"allowed": words[:0]}, {"allowed": words, "allowed_rows": vec(torch.int32)}):
        assert ops.process_logits(z, **rules, **masks).shape == (0, V)
        for draw in ({}, {"temperature": 1.0, "uniforms": torch.zeros(0, V, device=DEV)},
                     {"temperature": vec(torch.float32), "uniforms": vec(torch.float32)}):
            tok, logp = ops.choose_tokens(z, **rules, **masks, **draw)
            assert tok.shape == logp.shape == (0,) and tok.dtype == torch.long
    ids, flags = vec(torch.long), torch.zeros(V, dtype=torch.bool, device=DEV)
    for draw in ({}, {"temperature": 1.0, "uniforms": torch.zeros(0, T, device=DEV)},
                 {"temperature": 1.0, "uniforms": torch.zeros(0, T, V, device=DEV), "gumbel": True}):
        ops.choose_update(z, rules["bias"], flags, flags, 4, ids, ids, ids, ids, None, rules["history"], vec(torch.int32),
                          vec(torch.int32), None, 2, 0, repetition=1.2, allowed=words, token_rows=torch.zeros(V, dtype=torch.int32, device=DEV),
                          logp_out=torch.zeros(0, T, device=DEV), **draw)
    with pytest.raises(AssertionError):
        ops.process_logits(torch.zeros(2, V, device=DEV), allowed=words[:0])
