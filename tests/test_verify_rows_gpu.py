"""verify_drafts on rows that are cut over the blocks of a cluster: the first of equal largest logits, what is not finite in one block's part only."""

import numpy as np
import pytest
import torch

from test_verify_gpu import check, ints, make, ops  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("seqs,drafts,vocab", [(1, 4, 131071), (3, 0, 65537), (17, 2, 32000), (200, 1, 4099), (1, 0, 262145), (5, 3, 8192), (5, 3, 8191), (90, 5, 20011)])
def test_sizes_at_temperature_0(ops, dtype, seqs, drafts, vocab):  # noqa: F811
    rows = seqs * (drafts + 1)
    x, y, ids, u = make(rows, vocab, dtype, vocab, True, peaks=6)
    off = [i * (drafts + 1) for i in range(seqs + 1)]
    best = x.float().argmax(1)
    ids[1:] = torch.where(torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda()[1:] < 0.7, best[:-1], ids[1:])  # (some stand)
    check(ops, x, None, ids, u, off, 0.0)
    check(ops, x, y, ids, u, off, 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead", [0, 1, 5])
@pytest.mark.parametrize("rows,vocab", [(6, 131071), (6, 33000), (6, 16400), (6, 8200), (700, 33000), (1500, 33000)])
def test_equal_largest_logits_in_different_blocks(ops, dtype, lead, rows, vocab):  # noqa: F811
    """2, 4 and 8 blocks a row, rows at any address: pieces of 16 bytes go to the blocks in turn, so equals a piece, a block and the whole row apart."""
    wide = torch.zeros(rows, vocab + 9, device="cuda", dtype=dtype)
    x = wide[:, lead:lead + vocab]
    r = np.random.default_rng(vocab + lead)
    first = []
    for i in range(rows):
        a = int(r.integers(0, vocab))
        step = int(r.choice([1, 4, 8, 512, 1024, 1025, 4096, 8192]))
        places = {a, min(a + step, vocab - 1), vocab - 1}
        first.append(min(places))
        x[i, list(places)] = 3.0
    ids = torch.zeros(rows, dtype=torch.int64, device="cuda")
    ids[1:] = torch.tensor(first[:-1])
    u = torch.zeros(rows, 2, device="cuda")
    accepted, follows = ops.verify_drafts(x, ids, u, row_offsets=ints([0, rows]), temperature=0.0)
    assert accepted.tolist() == [rows - 1] and follows.tolist() == [first[-1]]
    ids[3] += 1
    accepted, follows = ops.verify_drafts(x, ids, u, row_offsets=ints([0, rows]), temperature=0.0)
    assert accepted.tolist() == [2] and follows.tolist() == [first[2]]


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("vocab", [131071, 9000])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_is_not_finite_in_one_block(ops, temperature, vocab, value):  # noqa: F811
    x, y, ids, u = make(24, vocab, torch.float32, 31, True, peaks=6)
    for i, at in ((1, 0), (5, 3), (9, 700), (13, vocab - 1), (17, vocab // 2)):
        x[i, at] = value
    y[20, 1234] = value
    off = [4 * i for i in range(7)]
    check(ops, x, y, ids, u, off, temperature)
    check(ops, x, None, ids, u, off, temperature)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_blocks_without_a_finite_logit(ops, temperature):  # noqa: F811
    """All but a few neighbours of a long row are -infinity: most blocks have nothing."""
    vocab = 100003
    x, y, ids, u = make(12, vocab, torch.float32, 32, True)
    for i in range(12):
        a = i * 9001 % (vocab - 9)
        keep = x[i, a:a + 3].clone()
        x[i] = -float("inf")
        x[i, a:a + 3] = keep
        if i:
            ids[i] = (i - 1) * 9001 % (vocab - 9) + 1
    check(ops, x, None, ids, u, [3 * i for i in range(5)], temperature, margin=False)
    check(ops, x, y, ids, u, [3 * i for i in range(5)], temperature, margin=False)
