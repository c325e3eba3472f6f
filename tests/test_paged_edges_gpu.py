"""kv_append and prefix_attention at the edges of their arguments: tables without rows, offsets in front of the call's rows, scores that are
large numbers, tables whose rows are one row.

Tolerances are those of test_paged_gpu.py; where nothing is rounded the results are compared bit by bit."""

import numpy as np
import pytest
import torch

from oracle import paged as P
from test_paged_gpu import check_append, check_attention, f64, ints, make_cache, ops  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ rotary


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_with_an_empty_rotary_table_leaves_everything_out(ops, interleaved):  # noqa: F811
    """No position is in the table: nothing is stored, queries are zero.  (No table at all: nothing is rotated.)"""
    k_pages, v_pages = make_cache(4, 16, 2, 64)
    old = k_pages.clone(), v_pages.clone()
    k, q = torch.randn(3, 2, 64, device="cuda").bfloat16(), torch.randn(3, 4, 64, device="cuda").bfloat16()
    out = ops.kv_append(k, k, k_pages, v_pages, ints([[0], [1], [2]]), ints([0, 3, 15]), q=q, rotary=torch.zeros(0, 64, device="cuda"), interleaved=interleaved)
    out2 = ops.kv_append(k, k, k_pages, v_pages, ints([[0], [1], [2]]), ints([0, 3, 15]), q=q, rotary=ops.rotary_table(9, 32)[:0])
    torch.cuda.synchronize()
    assert not out.any() and not out2.any() and torch.equal(k_pages, old[0]) and torch.equal(v_pages, old[1])


# ------------------------------------------------------------------------------------------------ offsets


def test_append_rows_between_sound_offsets_arrive(ops):  # noqa: F811
    """Sequence 1 has rows 0 to 3 as its tokens 5 to 8 (its offset is 5 rows in front of the call), sequence 2 the rest; the offsets around them
    make no sense."""
    k_pages, v_pages = make_cache(8, 16, 2, 64)
    want = k_pages.clone(), v_pages.clone()
    k, v, q = (torch.randn(12, 2, 64, device="cuda").bfloat16() for _ in range(3))
    for cache, x in zip(want, (k, v)):
        cache[1, 5:9], cache[2, 0:8] = x[:4], x[4:]
    q_out = torch.full_like(q, float("nan"))
    ops.kv_append(k, v, k_pages, v_pages, ints([[0], [1], [2]]), ints([0, 0, 0]), q=q, row_offsets=ints([2 ** 31 - 1, -5, 4, 2 ** 31 - 1]), q_out=q_out)
    torch.cuda.synchronize()
    assert torch.equal(q_out, q) and torch.equal(k_pages, want[0]) and torch.equal(v_pages, want[1])


@pytest.mark.parametrize("rows_of,first", [([4, 3, 6], -3), ([4, 3, 6], -6), ([40, 0, 9], -17)])
def test_append_offsets_in_front_of_the_rows(ops, rows_of, first):  # noqa: F811
    check_append(ops, rows_of=rows_of, lengths=[2, 15, 0], first_row=first, last_rows=2, starts=[3, 0, 9])


@pytest.mark.parametrize("heads,kv,d,rows_of,lengths,first", [
    (8, 8, 64, [4, 3, 6], [5, 9, 0], -3), (8, 2, 128, [4, 3, 6], [5, 70, 0], -6),          # few rows
    (16, 1, 64, [7, 5, 6], [30, 0, 90], -4), (16, 1, 128, [7, 5, 6], [30, 200, 9], -9),    # more
    (2, 2, 64, [200, 150], [0, 40], -30), (8, 2, 128, [90, 60, 70], [300, 0, 11], -110)])  # prompts
@pytest.mark.parametrize("prefix", [(), (150,)])
def test_attention_offsets_in_front_of_the_rows(ops, heads, kv, d, rows_of, lengths, first, prefix):  # noqa: F811
    """The first rows of a run that the call does not have count as tokens in front of those that it has."""
    torch.empty(2 ** 26, dtype=torch.float32, device="cuda").fill_(float("nan"))  # (what scratch may be given)
    check_attention(ops, lengths=lengths, rows_of=rows_of, prefix=prefix, heads=heads, kv=kv, d=d, first_row=first, last_rows=2)


def test_offsets_as_far_in_front_as_there_are_numbers(ops):  # noqa: F811
    """Tokens behind 2^31 others: beyond the table, at positions that `starts` brings back."""
    k_pages, v_pages = make_cache(4, 16, 2, 64)
    old = k_pages.clone()
    q, k = torch.randn(2, 4, 64, device="cuda").bfloat16(), torch.randn(2, 2, 64, device="cuda").bfloat16()
    off, t, n = [-2 ** 31, 2], ints([[2, 1]]), ints([0])
    rot = ops.rotary_table(9, 64)
    plain = ops.kv_append(k, k, k_pages, v_pages, t, n, q=q, row_offsets=ints(off))
    turned = ops.kv_append(k, k, k_pages, v_pages, t, n, q=q, row_offsets=ints(off), rotary=rot, starts=ints([-2 ** 31 + 5]))
    got = ops.prefix_attention(q, k_pages, v_pages, t, n, row_offsets=ints(off))
    torch.cuda.synchronize()
    assert torch.equal(k_pages, old) and torch.equal(plain, q)
    # rows 0 and 1 are tokens 2^31 and 2^31 + 1 at positions 5 and 6
    want = np.stack([P.rotate(x, f64(rot)[5 + i], False) for i, x in enumerate(f64(q))])
    assert (np.abs(f64(turned) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -22 * 12).all()
    want, width = P.prefix_attention_ref(f64(q), f64(k_pages), f64(v_pages), np.array([[2, 1]]), np.array([0]), row_offsets=np.array(off))
    assert (np.abs(f64(got) - want) <= 2.0 ** -8 * (np.abs(want) + width) + 2.0 ** -13 * width).all()


# ------------------------------------------------------------------------------------------------ scores


@pytest.mark.parametrize("heads,kv,d,n,tokens,length,prefix", [
    (4, 4, 64, 2, 3, 37, 90), (8, 8, 128, 2, 1, 61, 120),      # few rows
    (16, 1, 64, 2, 5, 70, 130), (16, 1, 128, 2, 5, 70, 130),   # more, two streams of items
    (16, 1, 64, 5, 7, 10, 200),                                # pairs over the prefix
    (2, 2, 64, 2, 140, 20, 100), (8, 2, 128, 2, 40, 60, 300)])  # pairs, prefix and own tokens in a row
@pytest.mark.parametrize("sign,low", [(1.0, 32), (-1.0, 32), (1.0, 26), (-1.0, 26), (1.0, 14)])
def test_attention_scores_that_are_large_numbers(ops, heads, kv, d, n, tokens, length, prefix, sign, low):  # noqa: F811
    """Scores of 2^low to 2^(low + 6), exact in fp32 and so far apart that the largest takes all of the weight: the result is its value, bit by
    bit where the scores are as large as that."""
    ps, own = 16, length + tokens
    width, pw = -(-own // ps), -(-prefix // ps)
    table, ptable = np.arange(n * width).reshape(n, width), n * width + np.arange(pw)[None]
    k_pages, v_pages = make_cache(n * width + pw, ps, kv, d)
    keys = prefix + n * own
    rank = np.stack([np.random.default_rng(c).permutation(keys) for c in range(d)])            # [d, keys]
    value = (128 + rank % 128) * 2.0 ** (rank // 128 + low - 24)                                    # ascending with the rank, eight bits
    ids = np.concatenate([ptable[0][np.arange(prefix) // ps] * ps + np.arange(prefix) % ps] +
                         [table[s][np.arange(own) // ps] * ps + np.arange(own) % ps for s in range(n)])
    flat = k_pages.view(-1, kv, d)
    flat[torch.from_numpy(ids).cuda()] = torch.from_numpy(np.ascontiguousarray(value.T))[:, None].expand(keys, kv, d).to("cuda", torch.bfloat16)
    rows = n * tokens
    column = np.arange(rows * heads).reshape(rows, heads) % d
    q = torch.zeros(rows, heads, d)
    q.scatter_(2, torch.from_numpy(column)[..., None], sign * 2.0 ** 20)
    off = np.arange(n + 1) * tokens
    got = ops.prefix_attention(q.cuda().bfloat16(), k_pages, v_pages, ints(table), ints([length] * n), ints(ptable), ints([prefix]), row_offsets=ints(off), scale=0.125)
    values = f64(v_pages).reshape(-1, kv, d)[ids]
    want = np.empty((rows, heads, d))
    for r in range(rows):
        s, i = divmod(r, tokens)
        seen = np.concatenate([np.arange(prefix), prefix + s * own + np.arange(length + i + 1)])
        for h in range(heads):
            best = seen[(sign * rank[column[r, h]][seen]).argmax()]
            want[r, h] = values[best, h // (heads // kv)]
    got = f64(got)
    assert (np.abs(got - want) <= (0.0 if low == 32 else 2.0 ** -7 + 2.0 ** -13) * np.abs(want)).all(), f"{(got != want).any(-1).sum()} of {rows * heads} rows differ, {np.isnan(got).any(-1).sum()} NaN"


# ------------------------------------------------------------------------------------------------ tables


def test_tables_whose_rows_are_one_row(ops):  # noqa: F811
    """Expanded tables: every sequence on the same pages, every group with the same prefix, every position with the same angles."""
    k_pages, v_pages = make_cache(6, 16, 2, 64)
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    t, p, n, m = ints([[0, 1]]).expand(3, 2), ints([[2, 3]]).expand(3, 2), ints([3, 9, 20]), ints([25]).expand(3)
    want = ops.prefix_attention(q, k_pages, v_pages, t.contiguous(), n, p.contiguous(), m.contiguous())
    assert torch.equal(ops.prefix_attention(q, k_pages, v_pages, t, n, p, m), want)
    one = ints([[4]]).expand(3, 1)
    want = ops.prefix_attention(q, k_pages, v_pages, one.contiguous(), ints([3, 9, 2]))
    assert torch.equal(ops.prefix_attention(q, k_pages, v_pages, one, ints([3, 9, 2])), want)
    rot = ops.rotary_table(9, 64)[4:5].expand(30, 64)
    k = torch.randn(3, 2, 64, device="cuda").bfloat16()
    caches = [(k_pages.clone(), v_pages.clone()) for _ in range(2)]
    a = ops.kv_append(k, k, *caches[0], t, n, q=q, rotary=rot)
    b = ops.kv_append(k, k, *caches[1], t.contiguous(), n, q=q, rotary=rot.contiguous())
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(*caches))
    assert not torch.equal(caches[0][0], k_pages)


# ------------------------------------------------------------------------------------------------ launches


def kernels(call):
    """Kernel nodes of a graph that the call is captured into."""
    from cuda.bindings import runtime as rt

    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    _, _, n = rt.cudaGraphGetNodes(rt.cudaGraph_t(graph.raw_cuda_graph()), 0)
    _, nodes, n = rt.cudaGraphGetNodes(rt.cudaGraph_t(graph.raw_cuda_graph()), n)
    kinds = [rt.cudaGraphNodeGetType(x)[1] for x in nodes[:n]]
    return sum(k == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds)


@pytest.mark.parametrize("heads,kv,n,tokens,prefix", [(4, 4, 3, 1, 90), (4, 4, 3, 0, 90), (2, 2, 2, 140, 90), (16, 1, 40, 1, 300), (16, 1, 2, 5, 130), (16, 1, 5, 7, 200)])
@pytest.mark.parametrize("native", [True, False])
def test_launches_are_counted(ops, monkeypatch, heads, kv, n, tokens, prefix, native):  # noqa: F811
    rows, pw = n * tokens, -(-prefix // 16)
    k_pages, v_pages = make_cache(n * 10 + pw, 16, kv, 64)
    t, p = ints(np.arange(n * 10).reshape(n, 10)), ints(n * 10 + np.arange(pw)[None])
    q, k = torch.randn(rows, heads, 64, device="cuda").bfloat16(), torch.randn(rows, kv, 64, device="cuda").bfloat16()
    lengths, off, m = ints([9] * n), ints(np.arange(n + 1) * tokens), ints([prefix])
    ops.kv_append(k, k, k_pages, v_pages, t, lengths, row_offsets=off)  # (the native host path is there)
    if not native:
        class Declines:
            kv_append = prefix_attention = staticmethod(lambda *a: None)
            launches = staticmethod(lambda: 0)
            reset_launches = staticmethod(lambda: None)

        monkeypatch.setattr(ops, "_native", Declines)
    for call in (lambda: ops.kv_append(k, k, k_pages, v_pages, t, lengths, row_offsets=off), lambda: ops.prefix_attention(q, k_pages, v_pages, t, lengths, p, m, row_offsets=off)):
        before = ops.launch_count()
        call()
        counted = ops.launch_count() - before
        assert counted == kernels(call)
