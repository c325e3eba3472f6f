"""prefix_attention over a cache in 4 bits at random sizes, and at those where another kernel, another cut or another path takes the call; tolerances as in
test_fp4_cache_gpu.py."""

import random

import numpy as np
import pytest
import torch

from test_fp4_cache_gpu import attend, check_append, ints, ops, pages_of  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(48))
def test_random_calls(ops, seed):  # noqa: F811
    r = random.Random(seed)
    heads, kv, d = r.choice(((8, 8, 64), (16, 4, 64), (4, 1, 64), (32, 8, 128), (12, 4, 128), (20, 2, 128), (3, 3, 128), (40, 1, 64)))
    groups = r.choice((0, 1, 1, 2, 5))
    n = (groups or 1) * r.choice((1, 2, 3, 7))
    tokens = r.choice(([1], [1], [1, 2, 3, 5], [0, 1, 4, 9], [0, 30, 70], [129, 2, 64], [260, 1]))
    rows_of = [r.choice(tokens) for _ in range(n)]
    lengths = [r.choice((0, 1, r.randrange(0, 60), r.randrange(0, 700), -1 if n > 2 else 3)) for _ in range(n)]
    single = all(t == 1 for t in rows_of) and r.random() < 0.7
    prefix = [r.choice((0, 1, 15, 16, 17, 127, 128, 129, r.randrange(1, 1500))) for _ in range(groups)] if groups else None
    ragged = groups > 1 and r.random() < 0.5
    sizes = None
    if ragged:
        cuts = sorted(r.randrange(0, n + 1) for _ in range(groups - 1))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [n])]

    def edit(table, pt):
        for t in (table, pt) if pt is not None else (table,):
            for i in range(t.shape[0]):
                for j in range(t.shape[1]):
                    if r.random() < 0.05:
                        t[i, j] = r.choice((-1, 10 ** 6, -(2 ** 31)))

    attend(ops, lengths=lengths, rows_of=rows_of, heads=heads, kv=kv, d=d, ps=r.choice((16, 32, 48, 128)), prefix=prefix, sizes=sizes, group_offsets=ragged, seed=seed,
           offsets=not single, first_row=0 if single else r.choice((0, 0, 3)), last_rows=0 if single else r.choice((0, 5)), width=r.choice((0, 0, 3, 40)),
           edit=edit if r.random() < 0.4 else None, any_bytes=False, shift=r.choice((0, 0, 3)))


@pytest.mark.parametrize("heads,kv,d", [(8, 8, 64), (32, 8, 128)])
@pytest.mark.parametrize("n,length", [(1, 1023), (1, 1024), (1, 1040), (3, 2500), (20, 1000), (19, 700), (80, 300), (75, 20)])
def test_where_one_launch_takes_a_call_and_where_not(ops, heads, kv, d, n, length):  # noqa: F811
    attend(ops, lengths=[max(0, length - 7 * i) for i in range(n)], rows_of=[1] * n, heads=heads, kv=kv, d=d, ps=16, offsets=False, seed=n)


@pytest.mark.parametrize("prefix", [[1], [15], [16], [31], [400]])
@pytest.mark.parametrize("first,last", [(0, 0), (2, 0), (0, 3), (5, 4)])
def test_one_launch_over_prefix_and_own_tokens(ops, prefix, first, last):  # noqa: F811
    """Ends of the prefix inside a unit, tokens of a call among themselves, rows in front of the first sequence and behind the last."""
    _, _, out = attend(ops, lengths=[0, 14, 16, -1, 100], rows_of=[2, 1, 4, 2, 3], heads=8, kv=4, d=64, ps=16, prefix=prefix, first_row=first, last_rows=last, seed=1)
    assert not out[:first].any() and not out[out.shape[0] - last:].any()


@pytest.mark.parametrize("d,rows", [(64, [40, 0, 90]), (128, [33, 17, 64]), (64, [300, 5, 200]), (128, [129, 140])])
def test_prompts_over_long_prefixes(ops, d, rows):  # noqa: F811
    attend(ops, lengths=[3] * len(rows), rows_of=rows, heads=4, kv=1, d=d, ps=32, prefix=[2500], seed=2)


def test_many_groups_of_uneven_sizes(ops):  # noqa: F811
    r = random.Random(7)
    sizes = [r.choice((0, 1, 5, 12, 40)) for _ in range(25)]
    n = sum(sizes)
    attend(ops, lengths=[r.randrange(0, 50) for _ in range(n)], rows_of=[1] * n, heads=8, kv=2, d=64, ps=16, prefix=[r.randrange(0, 900) for _ in sizes], sizes=sizes,
           group_offsets=True, offsets=False, seed=3)


def test_routes_agree(ops):  # noqa: F811
    """The native path of the call and the general one give the same bits; results do not depend on what scratch held."""
    args, kw, out = attend(ops, lengths=[50, 7, 0, 90], rows_of=[3, 1, 20, 150], heads=8, kv=2, d=128, ps=16, prefix=[1300], seed=4)
    assert torch.equal(ops.prefix_attention(*args, **{**kw, "k_scale": 1}), out)
    junk = torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")
    del junk
    assert torch.equal(ops.prefix_attention(*args, **kw), out)


def test_rows_of_other_sequences_change_nothing(ops):  # noqa: F811
    """A sequence alone and among others: the same within rounding, though another kernel may take it."""
    kv, d, ps = 2, 64, 16
    kp, vp = (torch.from_numpy(pages_of(60, ps, kv, d, i)).cuda() for i in range(2))
    table = ints(np.arange(60).reshape(4, 15).tolist())
    q = torch.randn(4, 8, d, device="cuda").bfloat16()
    lengths = ints([200, 100, 30, 5])
    out = ops.prefix_attention(q, kp, vp, table, lengths)
    for i in range(4):
        one = ops.prefix_attention(q[i:i + 1], kp, vp, table[i:i + 1], lengths[i:i + 1])
        assert (one.double() - out[i:i + 1].double()).abs().max() <= 2.0 ** -7 * out.double().abs().max()


@pytest.mark.parametrize("seed", range(12))
def test_random_appends(ops, seed):  # noqa: F811
    r = random.Random(100 + seed)
    n = r.randrange(1, 9)
    d = r.choice((16, 64, 80, 128, 256))
    check_append(ops, rows_of=[r.choice((0, 1, 2, 17, 130)) for _ in range(n)], lengths=[r.choice((0, 1, 15, 16, 33, 400, -1)) for _ in range(n)], heads=r.choice((1, 4, 6)), kv=r.choice((1, 2, 3)), d=d,
                 ps=r.choice((16, 48, 64)), rot=r.choice((0, 16, d)), dtype=r.choice((torch.bfloat16, torch.float32)), interleaved=r.random() < 0.5, shift=r.choice((0, 5)),
                 first_row=r.choice((0, 2)), last_rows=r.choice((0, 3)), seed=seed, k_scale=2.0 ** r.randrange(-3, 4), v_scale=2.0 ** r.randrange(-3, 4))
