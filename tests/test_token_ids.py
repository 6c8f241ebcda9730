"""Token ids of the teacher-forced forwards (Basecaller.hidden / logits, train_logits): negative ones count from the
vocabulary's end, as they do in an index; what is no id is refused where it can be seen without waiting for the device."""

import pytest
import torch

from viktor_amd.model import token_ids
from viktor_amd.synthetic import frames as synth_frames, make_model

DEV = "cuda"


@pytest.mark.parametrize("dt", [torch.int64, torch.int32])
def test_ids_as_an_index_takes_them(dt):
    """table[ids] is what F.embedding of the returned ids gives, for every id that an index takes; the caller's tensor stays."""
    V = 7
    table = torch.randn(V, 3, generator=torch.Generator().manual_seed(1))
    ids = torch.arange(-V, V).to(dt).view(2, V).t()  # (not contiguous)
    was = ids.clone()
    got = token_ids(ids, V, torch.device("cpu"))
    assert got.dtype == torch.int64 and got.is_contiguous() and got.shape == ids.shape
    assert torch.equal(torch.nn.functional.embedding(got, table), table[ids]) and torch.equal(ids, was)
    assert token_ids(ids[:0], V, torch.device("cpu")).shape == (0, 2)


def test_what_is_no_id_is_refused():
    cpu = torch.device("cpu")
    for bad in (torch.tensor([[0, 7]]), torch.tensor([[-8, 0]]), torch.tensor([[2 ** 32]])):
        with pytest.raises(IndexError):
            token_ids(bad, 7, cpu)
    for dt in (torch.float32, torch.bool, torch.complex64):
        with pytest.raises(IndexError):
            token_ids(torch.zeros(2, 3, dtype=dt), 7, cpu)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 2])
def test_negative_ids_in_scoring(group):
    """The logits of ids - V are those of the ids, from host and device tensors; ids past the ends are refused on the host."""
    m = make_model(1, n_layers=2, seed=3, norm_jitter=0.1, bias_jitter=0.1).to(DEV)
    fr = synth_frames(2, 64, 512, seed=4).to(DEV).repeat_interleave(group, 0)
    V, B = m.tokenizer.vocab_size, fr.shape[0]
    ids = torch.randint(0, V, (B, 128), generator=torch.Generator().manual_seed(5))
    neg = torch.where(torch.arange(128) % 3 == 0, ids - V, ids)
    with torch.no_grad():
        want = m.logits(fr, ids.to(DEV), group_size=group)
        for t in (ids, neg, neg.to(DEV), neg.int().to(DEV)):
            assert torch.equal(m.logits(fr, t, group_size=group), want)
        with pytest.raises(IndexError):
            m.logits(fr, ids + V, group_size=group)
        with pytest.raises(IndexError):
            m.logits(fr, ids.float().to(DEV), group_size=group)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 2])
def test_negative_ids_in_the_update(group):
    """train_logits and the embedding's gradient: those of the ids that the negative ones name."""
    from viktor_amd import train as TR
    m = make_model(1, n_layers=1, seed=6, norm_jitter=0.1, bias_jitter=0.1).to(DEV)
    fr = synth_frames(2, 64, 512, seed=7).to(DEV).repeat_interleave(group, 0)
    V, B = m.tokenizer.vocab_size, fr.shape[0]
    ids = torch.randint(0, V, (B, 64), generator=torch.Generator().manual_seed(8))
    neg = torch.where(torch.arange(64) % 3 == 0, ids - V, ids)
    emb = m.decoder.embed.weight
    seen = []
    for t in (ids.to(DEV), neg.to(DEV), neg):
        emb.grad = None
        z = TR.train_logits(m, fr, t, group_size=group)
        z.float().square().sum().backward()
        seen.append((z.detach(), emb.grad.clone()))
    for z, g in seen[1:]:
        assert torch.equal(z, seen[0][0]) and torch.equal(g, seen[0][1])
    with pytest.raises(IndexError):
        TR.train_logits(m, fr, ids + V, group_size=group)
