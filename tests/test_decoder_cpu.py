"""What the decoder refuses on the host, without a device: the blocks are replaced, pages and lengths are tensors on the CPU."""

import pytest
import torch

from velox_voice_b200 import decoder as D


@pytest.fixture
def dec():
    """A decoder of 64 positions and 40 pages of four tokens, whose blocks only say how many rows they were given."""
    d = object.__new__(D.HypothesisDecoder)
    d.cfg = D.DecoderConfig(blocks=1, d_model=64, heads=1, kv_heads=1, page_size=4, positions=64)
    d.k_pages = torch.zeros(1, 40, 4, 1, 64)
    d._free = list(range(40))
    d.rows = []
    d.embed = torch.zeros(10, 64)
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
