"""verify_drafts against its definition in fp64 (oracle/verify.py).

Results are whole numbers and have to be equal.  A comparison in fp64 can fall either way within the error of its sides: exponentials and quotients of relative
2^-50, sums of up to 2^17 positive terms added in another order, 2^-36 at the very most.  No comparison of the cases here comes nearer than that (it is asserted, of the
oracle's margins alone)."""

import numpy as np
import pytest
import torch

from oracle import verify as V

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from velox_voice_b200 import ops as o

    return o


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def make(rows, vocab, dtype, seed, drafter, gain=2.0, peaks=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * gain
    if peaks:
        x.scatter_add_(1, torch.randint(vocab, (rows, peaks), generator=g, device="cuda"), 6.0 + torch.randn(rows, peaks, generator=g, device="cuda"))
    y = x + 0.4 * torch.randn(rows, vocab, generator=g, device="cuda")
    near = y - torch.log(-torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
    ids = torch.randint(vocab, (rows,), generator=g, device="cuda")
    ids[1:] = near.argmax(1)[:-1]
    return x.to(dtype), y.to(dtype) if drafter else None, ids, torch.rand(rows, 2, generator=g, device="cuda")


def check(ops, x, y, ids, u, offsets=None, temperature=1.0, margin=True):
    got = ops.verify_drafts(x, ids, u, draft_logits=y, row_offsets=None if offsets is None else ints(offsets), temperature=temperature)
    torch.cuda.synchronize()
    want = V.verify_ref(x.double().cpu().numpy(), ids.cpu().numpy(), u.double().cpu().numpy(), None if y is None else y.double().cpu().numpy(),
                        None if offsets is None else np.array(offsets), temperature)
    assert not margin or min([w[2] for w in want], default=1.0) > 2.0 ** -36
    assert all(t.dtype == torch.int32 for t in got)
    assert [(int(a), int(b)) for a, b in zip(*got)] == [w[:2] for w in want]
    return got


COUNTS = [5, 1, 9, 2, 0, 6, 1, 8, 3, 5, 5, 5]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 3.0, 0.0])
@pytest.mark.parametrize("vocab", [5538, 1000, 1, 2, 7, 8, 9, 33])
def test_ragged_batches(ops, dtype, drafter, temperature, vocab):
    off = [0] + list(np.cumsum(COUNTS))
    for seed in range(3):
        x, y, ids, u = make(off[-1], vocab, dtype, seed, drafter, peaks=3 if vocab > 10 else 0)
        check(ops, x, y, ids, u, off, temperature)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("seqs,drafts,vocab", [(1, 4, 131071), (3, 0, 65537), (17, 2, 32000), (200, 1, 4099), (1, 0, 262145)])
def test_sizes(ops, dtype, seqs, drafts, vocab):
    rows = seqs * (drafts + 1)
    x, y, ids, u = make(rows, vocab, dtype, vocab, True, peaks=6)
    check(ops, x, y, ids, u, [i * (drafts + 1) for i in range(seqs + 1)])


def test_rows_of_one_token_without_offsets(ops):
    x, _, ids, u = make(300, 777, torch.float32, 5, False)
    accepted, _ = check(ops, x, None, ids, u)
    assert not accepted.any()


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_strides_and_types_of_ids(ops, ids_dtype):
    x, y, ids, u = make(20, 501, torch.bfloat16, 6, True)
    wide, other = torch.zeros(20, 1009, dtype=torch.bfloat16, device="cuda"), torch.zeros(20, 777, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:504], other[:, 1:502] = x, y
    off = [0, 4, 5, 11, 20]
    a = check(ops, x, y, ids.to(ids_dtype), u, off)
    b = check(ops, wide[:, 3:504], other[:, 1:502], ids.to(ids_dtype), u, off)
    c = check(ops, x.t().contiguous().t(), y, ids.to(ids_dtype), torch.stack([u, u], 1)[:, 1], off)
    assert torch.equal(a[1], b[1]) and torch.equal(a[1], c[1])


def test_offsets_around_the_rows(ops):
    """Rows in front of the first sequence and behind the last, offsets outside."""
    x, y, ids, u = make(30, 300, torch.float32, 7, True)
    check(ops, x, y, ids, u, [3, 9, 9, 14, 22])
    check(ops, x, y, ids, u, [-4, 9, 14, 40])
    check(ops, x, y, ids, u, [30, 31, 99])


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_rows_without_probabilities(ops, temperature):
    inf = float("inf")
    x, y, ids, u = make(48, 200, torch.float32, 8, True)
    off = [4 * i for i in range(13)]
    x[1], x[4, 7], x[8, 3], x[15], x[19, 5] = -inf, float("nan"), inf, -inf, float("nan")
    y[21], y[24, 9], y[28, 1], y[35] = -inf, float("nan"), inf, float("nan")
    x[40:44, 50:], y[41, :60] = -inf, -inf
    x[44:48] = -inf
    x[44:48, 17] = 2.0
    check(ops, x, y, ids, u, off, temperature)
    check(ops, x, None, ids, u, off, temperature)


def test_ids_outside_the_vocabulary(ops):
    x, y, ids, u = make(12, 100, torch.bfloat16, 9, True)
    ids[1], ids[5], ids[7], ids[10] = -1, 100, 2 ** 40, -2 ** 50
    for y in (y, None):
        accepted, _ = check(ops, x, y, ids, u, [0, 4, 8, 12])
        assert int(accepted[0]) == 0


def test_the_ends_of_the_random_numbers(ops):
    """0 takes a draft of any probability and the first token with a weight; the largest below 1 the last tokens."""
    x, y, ids, u = make(40, 500, torch.float32, 10, True)
    off = [5 * i for i in range(9)]
    u[:20] = 0.0
    u[20:] = 1.0 - 2.0 ** -24
    x[::3, :7] = -float("inf")
    x[1::3, 400:] = -float("inf")
    check(ops, x, y, ids, u, off, margin=False)
    accepted, follows = ops.verify_drafts(x, ids, torch.ones_like(u), draft_logits=y, row_offsets=ints(off))  # (not below 1: still a token)
    assert (follows >= 0).all()


def test_equal_probabilities_stand(ops):
    """The drafter is the target: all drafts stand, whatever the numbers."""
    x, _, ids, u = make(60, 1500, torch.bfloat16, 11, True)
    off = [6 * i for i in range(11)]
    accepted, _ = check(ops, x, x.clone(), ids, u, off, margin=False)
    assert (accepted == 5).all()
    u[:, 0] = 1.0 - 2.0 ** -24
    accepted, _ = ops.verify_drafts(x, ids, u, draft_logits=x, row_offsets=ints(off))
    assert (accepted == 5).all()


def test_ties_go_to_the_first(ops):
    x = torch.zeros(6, 5000, device="cuda", dtype=torch.bfloat16)
    x[0, 4321], x[0, 77], x[1, 4999], x[2, 0] = 1, 1, 1, 1
    x[3] = -1
    off = [0, 2, 3, 6]
    for lead in (0, 1, 3):  # (rows that begin beside a 16-byte address)
        w = torch.zeros(6, 5003, device="cuda", dtype=torch.bfloat16)
        w[:, lead:lead + 5000] = x
        ids = ints([0, 77, 0, 0, 0, 0])
        accepted, follows = check(ops, w[:, lead:lead + 5000], None, ids, torch.zeros(6, 2, device="cuda"), off, 0.0)
        assert accepted.tolist() == [1, 0, 2] and follows.tolist() == [4999, 0, 0]


def test_drawn_tokens_have_their_probabilities(ops):
    """Drafts and what follows them together are distributed as the target: 40,000 draws over 12 tokens, each share within five standard deviations."""
    n, vocab = 40000, 12
    g = torch.Generator(device="cuda").manual_seed(0)
    x, y = torch.randn(vocab, generator=g, device="cuda"), torch.randn(vocab, generator=g, device="cuda")
    q = torch.softmax(y, 0)
    drafts = torch.multinomial(q, n, replacement=True, generator=g)
    ids = torch.stack([torch.zeros_like(drafts), drafts], 1).flatten()
    u = torch.rand(2 * n, 2, generator=g, device="cuda")
    accepted, follows = ops.verify_drafts(x.repeat(2 * n, 1), ids, u, draft_logits=y.repeat(2 * n, 1), row_offsets=torch.arange(n + 1, device="cuda", dtype=torch.int32) * 2)
    first = torch.where(accepted == 1, drafts, follows.long())
    p = torch.softmax(x.double(), 0)
    share = torch.bincount(first, minlength=vocab).double() / n
    assert ((share - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all()


def test_nothing_to_do(ops):
    x, _, ids, u = make(4, 50, torch.float32, 12, False)
    for off in ([2], [0, 0, 0], [4, 4]):
        a, b = ops.verify_drafts(x, ids, u, row_offsets=ints(off))
        assert a.tolist() == [0] * (len(off) - 1) and b.tolist() == [-1] * (len(off) - 1)
    a, b = ops.verify_drafts(x[:0], ids[:0], u[:0], row_offsets=ints([0, 0]))
    assert a.tolist() == [0] and b.tolist() == [-1]
    assert ops.verify_drafts(x[:0], ids[:0], u[:0])[0].numel() == 0


def test_in_graphs_and_on_a_side_stream(ops):
    x, y, ids, u = make(40, 5538, torch.bfloat16, 13, True)
    off = ints([5 * i for i in range(9)])
    want = ops.verify_drafts(x, ids, u, draft_logits=y, row_offsets=off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.verify_drafts(x, ids, u, draft_logits=y, row_offsets=off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want[1], got[1])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.verify_drafts(x, ids, u, draft_logits=y, row_offsets=off)
        graphs.append((g, out))
    for seed in range(3):
        for t, n in zip((x, y, ids, u), make(40, 5538, torch.bfloat16, 20 + seed, True)):
            t.copy_(n)
        for g, _ in graphs:
            g.replay()
        want = check(ops, x, y, ids, u, [5 * i for i in range(9)])
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals_and_launches(ops):
    x, y, ids, u = make(6, 50, torch.float32, 14, True)
    off = ints([0, 3, 6])
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1e-9), dict(draft_logits=y[:5]), dict(draft_logits=y.bfloat16()),
               dict(row_offsets=off.long()), dict(row_offsets=off[:0])):
        with pytest.raises(ValueError):
            ops.verify_drafts(x, ids, u, **{"row_offsets": off, **kw})
    for args in ((x[0], ids, u), (x, ids[:5], u), (x, ids.float(), u), (x, ids, u[:, :1]), (x, ids, u.double()), (x[:, :0], ids, u)):
        with pytest.raises(ValueError):
            ops.verify_drafts(*args, row_offsets=off)
    with pytest.raises(TypeError):
        ops.verify_drafts(x.half(), ids, u, row_offsets=off)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.verify_drafts(x, ids.cpu(), u, row_offsets=off)
    ops.reset_launch_count()
    ops.verify_drafts(x, ids, u, row_offsets=off, temperature=1)
    assert ops.launch_count() == 2


@pytest.mark.parametrize("temperature,level", [(0.01, 500.0), (0.01, -500.0), (2.0 ** -10, 64.0), (1.0, 30000.0), (2.0 ** -20, 0.25), (2.0 ** -20, -1.0)])
@pytest.mark.parametrize("drafter", [True, False])
def test_logits_that_are_large_for_their_temperature(ops, temperature, level, drafter):
    """The largest logit over the temperature is 30,000 to 1,000,000, and the uniform numbers are 2^-11 from where a draft falls."""
    x, y, ids, u = make(120, 3000, torch.float32, 21, True, gain=1.0)
    x, y = level + temperature * x, level + temperature * y
    p, q = (torch.softmax(t.double() / temperature, 1)[:-1].gather(1, ids[1:, None])[:, 0] for t in (x, y))
    side = torch.where(torch.arange(119, device="cuda") % 7 < 5, -1.0, 1.0)  # (five that stand, then two that fall)
    ratio = p / q if drafter else p
    u[:-1, 0] = (ratio * (1 + side * 2.0 ** -11)).clamp(0, 1 - 2.0 ** -24).float()
    check(ops, x, y if drafter else None, ids, u, [6 * i for i in range(21)], temperature)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [1.0, 0.5, 2.0 ** -20, 2.0 ** 20, 0.0])
def test_lowest_and_largest_logits(ops, dtype, temperature):
    """Tokens that are masked with the type's lowest value have no probability beside others, and one like another where they are all there is.
    (A masked draft has 0 on both sides of its comparison, of any rounding: no margin is asked for.)"""
    x, y, ids, u = make(32, 517, dtype, 22, True)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x[:8, 100:], y[:8, 90:] = low, low
    x[8:16], y[9] = low, low
    x[16:20, 5], x[20:24], y[21] = high, high, high
    x[24:28, 3:], x[24:28, :3] = low, -float("inf")
    off = [4 * i for i in range(9)]
    check(ops, x, y, ids, u, off, temperature, margin=False)
    check(ops, x, None, ids, u, off, temperature, margin=False)


@pytest.mark.parametrize("seqs,vocab", [(2, 2 ** 22 + 5), (150, 40001), (40, 70003)])
def test_draws_from_long_rows(ops, seqs, vocab):
    """Rows that a cluster or a block has alone, drawn from at their ends and between.  (A number of 0 asks for the first token that has a weight: tokens in front of it
    have none, at any rounding, so no margin is asked for.)"""
    x, y, ids, u = make(2 * seqs, vocab, torch.bfloat16, 23, True, peaks=0)
    u[0::2, 0] = 1 - 2.0 ** -24
    u[0::3, 1], u[1::5, 1] = 0.0, 1 - 2.0 ** -24
    check(ops, x, y, ids, u, [2 * i for i in range(seqs + 1)], margin=False)
