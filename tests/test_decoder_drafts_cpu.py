"""Drafts and the 4-bit cache of the decoder, on the host: what verify() leaves in lengths and counts, what is refused."""

import pytest
import torch

from velox_voice_b200 import decoder as D


@pytest.fixture
def dec(monkeypatch):
    """A decoder of 64 positions and 40 pages of 16 tokens, whose blocks only say how many rows they were given."""
    monkeypatch.setattr(D.ops, "ln_quantize", lambda x, *a: x)
    d = object.__new__(D.HypothesisDecoder)
    d.cfg = D.DecoderConfig(blocks=1, d_model=64, heads=1, kv_heads=1, page_size=16, positions=64, cache="fp4")
    d.k_pages = torch.zeros(1, 40, 1, 1, 576, dtype=torch.uint8)
    d._free = list(range(40))
    d.embed = torch.zeros(10, 64)
    d.after, d.head = (None, None), lambda x: x
    d._blocks = lambda x, *a, **k: x
    return d


def test_verify_keeps_the_drafts_that_stand(dec, monkeypatch):
    seen = {}

    def verify(logits, ids, uniforms, *, draft_logits, row_offsets, temperature):
        seen.update(logits=logits, ids=ids, offsets=row_offsets.tolist(), temperature=temperature)
        return torch.tensor([2, 0, 0, 3], dtype=torch.int32), torch.tensor([7, 8, -1, 9], dtype=torch.int32)

    monkeypatch.setattr(D.ops, "verify_drafts", verify)
    hyp = dec.begin(dec.read(torch.zeros(10, 64), [4, 6]), 2, 12)
    hyp.lengths[3] = -1
    ids = torch.arange(10)
    accepted, following = dec.verify(hyp, ids, [4, 2, 0, 4], torch.rand(10, 2), temperature=0.5)
    assert seen["offsets"] == [0, 4, 6, 6, 10] and seen["logits"].shape == (10, 64) and seen["temperature"] == 0.5
    assert hyp.lengths.tolist() == [3, 1, 0, -1] and following.tolist() == [7, 8, -1, 9]
    assert hyp.tokens == [4, 2, 0, 4]
    dec.settle(hyp)
    assert hyp.tokens == [3, 1, 0, 4]
    with pytest.raises(RuntimeError, match="room"):
        dec.verify(hyp, torch.zeros(10, dtype=torch.long), [10, 0, 0, 0], torch.rand(10, 2))
    dec.verify(hyp, torch.zeros(9, dtype=torch.long), [9, 0, 0, 0], torch.rand(9, 2))
    dec.release(hyp)
    with pytest.raises(RuntimeError, match="handed back"):
        dec.settle(hyp)


def test_a_refused_call_keeps_nothing(dec, monkeypatch):
    def refuse(*a, **k):
        raise ValueError("uniforms")

    monkeypatch.setattr(D.ops, "verify_drafts", refuse)
    hyp = dec.begin(dec.read(torch.zeros(10, 64), [4, 6]), 2, 12)
    hyp.lengths.copy_(torch.tensor([3, 0, -1, 5], dtype=torch.int32))
    hyp.tokens = [3, 0, 2, 5]
    with pytest.raises(ValueError, match="uniforms"):
        dec.verify(hyp, torch.arange(10), [4, 2, 4, 0], torch.rand(3, 2))
    assert hyp.lengths.tolist() == [3, 0, -1, 5] and hyp.tokens == [3, 0, 2, 5]


def test_unknown_caches_and_page_sizes_are_refused():
    for kw, text in ((dict(cache="fp5"), "cache"), (dict(cache="fp4", page_size=24), "16 n")):
        cfg = D.DecoderConfig(blocks=0, **kw)
        with pytest.raises(ValueError, match=text):
            d = object.__new__(D.HypothesisDecoder)
            _init_cache(d, cfg)


def _init_cache(d, cfg):
    """The part of the constructor that makes the pages, on the CPU."""
    import unittest.mock as mock

    with mock.patch.object(D, "PackedLinear", lambda *a: None), mock.patch.object(D.ops, "rotary_table", lambda *a, **k: None):
        d.__init__(cfg, D.make_weights(cfg), 4, device="cpu")
