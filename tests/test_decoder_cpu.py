"""What the decoder refuses on the host, without a device: the blocks are replaced, pages and lengths are tensors on the CPU."""

import pytest
import torch

from velox_voice_b200 import decoder as D


class Head:
    """Stands for the output layer."""

    def __call__(self, x):
        return x

    argmax = __call__


@pytest.fixture
def dec(monkeypatch):
    """A decoder of 64 positions and 40 pages of four tokens, whose blocks only say how many rows they were given."""
    monkeypatch.setattr(D.ops, "ln_quantize", lambda x, *a: x)
    d = object.__new__(D.HypothesisDecoder)
    d.cfg = D.DecoderConfig(blocks=1, d_model=64, heads=1, kv_heads=1, page_size=4, positions=64)
    d.k_pages = torch.zeros(1, 40, 4, 1, 64)
    d._free = list(range(40))
    d.rows = []
    d.embed = torch.zeros(10, 64)
    d.after, d.head = (None, None), Head()
    d._blocks = lambda x, *a, **k: (d.rows.append(x.shape[0]), x)[1]
    return d


def frames(n):
    return torch.zeros(n, 64)


def test_read_refuses_frames_beyond_the_positions(dec):
    """Rows at positions that the rotary table does not have are not stored: the pages would be attended as they were."""
    dec.read(frames(64), [64])
    with pytest.raises(ValueError, match="positions"):
        dec.read(frames(65), [65])
    with pytest.raises(ValueError, match="positions"):
        dec.read(frames(75), [5, 70])
    assert dec.rows == [64] and len(dec._free) == 40 - 16


def test_begin_refuses_tokens_beyond_the_positions(dec):
    utt = dec.read(frames(70), [10, 60])
    dec.begin(utt, 1, 4)
    with pytest.raises(ValueError, match="positions"):
        dec.begin(utt, 1, 5)
    assert len(dec._free) == 40 - 3 - 15 - 2


def test_step_refuses_tokens_beyond_the_room(dec):
    """A token without a page is not stored; the hypothesis would go on without it."""
    hyp = dec.begin(dec.read(frames(10), [4, 6]), 2, 3)
    ids = torch.zeros(4, dtype=torch.long)
    for _ in range(3):
        dec.step(hyp, ids)
    with pytest.raises(RuntimeError, match="room"):
        dec.step(hyp, ids)
    assert hyp.lengths.tolist() == [3] * 4 and dec.rows == [10, 4, 4, 4]


def test_score_refuses_tokens_beyond_the_room(dec):
    hyp = dec.begin(dec.read(frames(6), [6]), 3, 5)
    dec.step(hyp, torch.zeros(3, dtype=torch.long))
    dec.score(hyp, torch.zeros(6, dtype=torch.long), [4, 2, 0])
    assert hyp.lengths.tolist() == [5, 3, 1]
    with pytest.raises(RuntimeError, match="room"):
        dec.score(hyp, torch.zeros(4, dtype=torch.long), [0, 3, 1])
    dec.score(hyp, torch.zeros(3, dtype=torch.long), [0, 2, 1])
    with pytest.raises(RuntimeError, match="room"):
        dec.step(hyp, torch.zeros(3, dtype=torch.long))
    assert hyp.lengths.tolist() == [5, 5, 2]


def test_score_refuses_counts_that_do_not_fit_the_ids(dec):
    hyp = dec.begin(dec.read(frames(6), [6]), 3, 5)
    for ids, counts in ((6, [4, 2]), (6, [2, 2, 1]), (5, [2, 2, 2]), (4, [5, -1, 0])):
        with pytest.raises(ValueError, match="counts"):
            dec.score(hyp, torch.zeros(ids, dtype=torch.long), counts)
    assert hyp.lengths.tolist() == [0, 0, 0] and dec.rows == [6]


def test_pages_that_were_handed_back_are_not_used(dec):
    """They may be another owner's by then."""
    utt = dec.read(frames(6), [6])
    hyp, other = dec.begin(utt, 2, 5), dec.begin(utt, 1, 5)
    ids = torch.zeros(2, dtype=torch.long)
    dec.step(hyp, ids)
    dec.release(hyp)
    for call in (lambda: dec.step(hyp, ids), lambda: dec.score(hyp, ids, [1, 1]), lambda: dec.compile_step(hyp)):
        with pytest.raises(RuntimeError, match="handed back"):
            call()
    dec.release(utt)
    for call in (lambda: dec.step(other, ids[:1]), lambda: dec.score(other, ids[:1], [1]), lambda: dec.begin(utt, 1, 1)):
        with pytest.raises(RuntimeError, match="handed back"):
            call()
    dec.release(other)
    dec.release(other)
    assert sorted(dec._free) == list(range(40)) and dec.rows == [6, 2]


def test_begin_refuses_no_beams_and_negative_room(dec):
    utt = dec.read(frames(6), [6])
    for beams, tokens in ((0, 5), (-1, 5), (2, -1)):
        with pytest.raises(ValueError, match="beams"):
            dec.begin(utt, beams, tokens)
    assert len(dec._free) == 38


def test_a_read_that_fails_keeps_no_pages(dec):
    def fails(*a, **k):
        raise TypeError("frames of another type")

    dec._blocks = fails
    with pytest.raises(TypeError):
        dec.read(frames(30), [10, 20])
    assert sorted(dec._free) == list(range(40))
