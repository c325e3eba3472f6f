"""kv_append and prefix_attention against their definitions in fp64 (oracle/paged.py).

Tolerances, fixed by the number formats.  A stored or returned bf16 value is the nearest to an fp32 result: half a unit in the last
of 8 significant bits, at most 2^-8 of it.  The rotation's two products and their sum in fp32 add at most 2^-22 (|a| + |b|).  Attention rounds each
probability to bf16 (2^-8 of it, so 2^-8 sum_j w_j |v_j| of a result) and its result once; scores, exponentials and sums in fp32 change a
weight by less than 2^-13 at the scores used here (|s| < 60: fp32 products and sums of 128 terms, 2^-24 each, one rounding of
s log2 e, an exponential within 2^-22)."""

import numpy as np
import pytest
import torch

from oracle import paged as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from velox_voice_b200 import ops as o

    return o


def f64(t):
    return t.detach().cpu().double().numpy()


def ints(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def make_cache(pages, ps, kv, d, layout="tokens", fill=None, seed=0):
    """k_pages, v_pages [pages, ps, kv, d] in the given order of memory; `fill`: a value for every place instead of random ones"""
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    out = []
    for _ in range(2):
        if layout == "heads":   # heads outermost in a page
            t = torch.randn(pages, kv, ps, d, generator=g, device="cuda").bfloat16().transpose(1, 2)
        elif layout == "wide":  # a page is a part of a larger row
            t = torch.randn(pages, ps + 1, kv, d + 8, generator=g, device="cuda").bfloat16()[:, :ps, :, :d]
        else:
            t = torch.randn(pages, ps, kv, d, generator=g, device="cuda").bfloat16()
        if fill is not None:
            t.fill_(fill)
        out.append(t)
    return out


def tables(counts, total, seed=0, width=None):
    """page_table rows with `counts` pages each, from a shuffled pool; unused entries -1"""
    order = np.random.default_rng(seed).permutation(total)
    t = np.full((len(counts), max(max(counts), 1) if width is None else width), -1, dtype=np.int64)
    at = 0
    for i, c in enumerate(counts):
        t[i, :c] = order[at:at + c]
        at += c
    assert at <= total
    return t, order[at:]


# ------------------------------------------------------------------------------------------------ kv_append


def check_append(ops, *, rows_of, lengths, heads=4, kv=2, d=64, ps=16, rot=64, dtype=torch.bfloat16, interleaved=False, layout="tokens",
                 starts=None, positions=None, edit_table=None, offsets=True, first_row=0, last_rows=0, fused=True, seed=0, stream=None):
    n = len(lengths)
    rows = first_row + sum(rows_of) + last_rows
    off = np.cumsum([first_row] + list(rows_of))
    counts = [-(-(max(l, 0) + c) // ps) for l, c in zip(lengths, rows_of)]
    total = sum(counts) + 2
    table, _ = tables(counts, total, seed)
    if edit_table is not None:
        edit_table(table)
    k_pages, v_pages = make_cache(total, ps, kv, d, layout, seed=seed)
    before = k_pages.clone(), v_pages.clone()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, (heads + 2 * kv) * d + (0 if fused else 3), generator=g, device="cuda").to(dtype)
    if not fused:  # rows that do not start at multiples of 16 bytes
        x = x[:, 3:]
    q, k, v = x[:, :heads * d].unflatten(1, (heads, d)), x[:, heads * d:(heads + kv) * d].unflatten(1, (kv, d)), x[:, (heads + kv) * d:].unflatten(1, (kv, d))
    start = [0] * n if starts is None else starts
    last = max([s + max(l, 0) + c for s, l, c in zip(start, lengths, rows_of)] + [1])
    rotary = ops.rotary_table(last if positions is None else positions, rot) if rot else None
    kw = dict(q=q, rotary=rotary, interleaved=interleaved, row_offsets=ints(off) if offsets else None, starts=None if starts is None else ints(starts))
    q_out = ops.kv_append(k, v, k_pages, v_pages, ints(table), ints(lengths), **kw)
    torch.cuda.synchronize()
    want_q, want_k, want_v, stored = P.kv_append_ref(f64(q), f64(k), f64(v), f64(before[0]), f64(before[1]), table, np.array(lengths),
                                                     None if rotary is None else f64(rotary), interleaved, off if offsets else None, starts)
    assert q_out.dtype == torch.bfloat16
    for got, want in ((q_out, want_q), (k_pages, want_k), (v_pages, want_v)):
        assert (np.abs(f64(got) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -22 * 12).all()
    # what no token was written to is as it was, bit for bit
    keep = torch.from_numpy(~stored).cuda()
    for got, old in zip((k_pages, v_pages), before):
        assert torch.equal(got[keep].view(torch.int16), old[keep].view(torch.int16))
    return q_out, stored


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,d,rot,ps", [(8, 8, 64, 64, 16), (32, 8, 128, 128, 64), (6, 2, 128, 64, 24), (4, 1, 256, 16, 1), (3, 3, 16, 16, 7), (5, 5, 80, 48, 16), (4, 2, 64, 0, 16)])
def test_append_single_tokens(ops, dtype, interleaved, heads, kv, d, rot, ps):
    lengths = [0, 1, ps - 1, ps, ps + 1, 5 * ps + 3, 200]
    check_append(ops, rows_of=[1] * 7, lengths=lengths, heads=heads, kv=kv, d=d, rot=rot, ps=ps, dtype=dtype, interleaved=interleaved, offsets=False)


@pytest.mark.parametrize("layout", ["tokens", "heads", "wide"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_ragged_rows(ops, layout, dtype):
    check_append(ops, rows_of=[5, 0, 33, 1, 0, 200, 17], lengths=[0, 4, 15, 16, 9, 70, 1], layout=layout, dtype=dtype, starts=[0, 3, 375, 0, 1, 12, 9], seed=3)


@pytest.mark.parametrize("rows", [1, 2, 3000, 9001])
def test_append_one_long_sequence(ops, rows):
    check_append(ops, rows_of=[rows], lengths=[3], heads=2, kv=1, seed=rows, dtype=torch.float32)


def test_append_leaves_out_what_has_no_place(ops):
    """Rows of no sequence, inactive sequences, dropped pages, ids that are no pages, more tokens than the table holds."""
    def edit(t):
        t[0, 1] = -1
        t[2, 0] = 10 ** 6
        t[3, :] = -(2 ** 31)

    q_out, stored = check_append(ops, rows_of=[40, 9, 20, 5, 12], lengths=[0, -1, 3, 0, -2 ** 31], edit_table=edit, first_row=3, last_rows=6, seed=5)
    assert not f64(q_out[:3]).any() and not f64(q_out[43:52]).any() and not f64(q_out[-6:]).any()
    assert stored.sum() == 24 + 20 - 13


def test_append_positions_beyond_the_rotary_table(ops):
    q_out, stored = check_append(ops, rows_of=[10, 10, 10], lengths=[0, 0, 0], starts=[0, 25, -4], positions=30, seed=6)
    assert stored.sum() == 10 + 5 + 6


def test_append_lengths_beyond_the_table(ops):
    """Lengths up to the largest integer: no place, no fault."""
    k_pages, v_pages = make_cache(4, 16, 2, 64)
    old = k_pages.clone()
    k = torch.randn(3, 2, 64, device="cuda").bfloat16()
    t = ints([[0, 1]] * 3)
    out = ops.kv_append(k, k, k_pages, v_pages, t, ints([32, 10 ** 6, 2 ** 31 - 1]), q=k, rotary=None)
    torch.cuda.synchronize()
    assert torch.equal(k_pages, old) and torch.equal(out, k)


def test_append_offsets_that_do_not_ascend(ops):
    """Offsets that make no sense store nothing outside the cache; rows between sound ones still arrive."""
    k_pages, v_pages = make_cache(8, 16, 2, 64)
    k = torch.randn(12, 2, 64, device="cuda").bfloat16()
    out = ops.kv_append(k, k, k_pages, v_pages, ints([[0], [1], [2]]), ints([0, 0, 0]), q=k, row_offsets=ints([2 ** 31 - 1, -5, 4, 2 ** 31 - 1]))
    torch.cuda.synchronize()
    assert torch.isfinite(out.float()).all()


def test_append_strided_misaligned_and_in_place(ops):
    check_append(ops, rows_of=[7, 9], lengths=[1, 2], fused=False, seed=8)
    check_append(ops, rows_of=[7, 9], lengths=[1, 2], fused=False, dtype=torch.float32, seed=8)
    k_pages, v_pages = make_cache(4, 16, 2, 64)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    k = torch.randn(2, 1, 64, device="cuda").bfloat16().expand(2, 2, 64)  # one head for both
    rot = ops.rotary_table(64, 64)
    want = ops.kv_append(k.contiguous(), k.contiguous(), k_pages.clone(), v_pages.clone(), ints([[0], [1]]), ints([3, 9]), q=q, rotary=rot)
    kept = q.data_ptr()
    got = ops.kv_append(k, k, k_pages, v_pages, ints([[0], [1]]), ints([3, 9]), q=q, rotary=rot, q_out=q)
    assert got.data_ptr() == kept and torch.equal(got, want)
    assert torch.equal(v_pages[1, 9], k[1])
    assert ops.kv_append(k, k, k_pages, v_pages, ints([[0], [1]]), ints([3, 9])) is None


def test_append_nothing(ops):
    k_pages, v_pages = make_cache(2, 16, 2, 64)
    e = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = ops.kv_append(e, e, k_pages, v_pages, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([]), q=e)
    assert out.shape == (0, 2, 64)
    # rows, but no sequence that they could belong to; sequences, but a cache without pages
    k = torch.ones(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = ops.kv_append(k, k, k_pages, v_pages, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([]), q=k, row_offsets=ints([0]))
    assert not out.any()
    none = torch.empty(0, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = ops.kv_append(k, k, none, none, torch.full((4, 0), -1, dtype=torch.int32, device="cuda"), ints([0] * 4), q=k)
    assert torch.equal(out, k)


# ------------------------------------------------------------------------------------------------ prefix_attention


def check_attention(ops, *, lengths, rows_of=None, prefix=(), sizes=None, heads=8, kv=8, d=64, ps=16, layout="tokens", spread=1.0, seed=0,
                    edit=None, edit_prefix=None, first_row=0, last_rows=0, extra_width=0, scale=None, equal_groups=False, lots=None):
    """Everything that no row may read holds NaN."""
    n = len(lengths)
    tokens = [1] * n if rows_of is None else list(rows_of)
    rows = first_row + sum(tokens) + last_rows
    off = np.cumsum([first_row] + tokens)
    counts = [-(-(max(l, 0) + t) // ps) for l, t in zip(lengths, tokens)]
    pcounts = [-(-p // ps) for p in prefix]
    total = sum(counts) + sum(pcounts) + 2 if lots is None else lots
    table, rest = tables(counts, total, seed, width=max(max(counts), 1) + extra_width)
    ptable = np.full((len(prefix), max(pcounts + [1]) + extra_width), -1, dtype=np.int64)
    at = 0
    for i, c in enumerate(pcounts):
        ptable[i, :c] = rest[at:at + c]
        at += c
    k_pages, v_pages = make_cache(total, ps, kv, d, layout, fill=float("nan"))
    g = torch.Generator(device="cuda").manual_seed(seed)
    for tab, lens in ((table, [max(l, 0) + t if l >= 0 else 0 for l, t in zip(lengths, tokens)]), (ptable, prefix)):
        for row, m in zip(tab, lens):
            for j in range(0, m, ps):
                c = min(ps, m - j)
                k_pages[row[j // ps], :c] = torch.randn(c, kv, d, generator=g, device="cuda").bfloat16()
                v_pages[row[j // ps], :c] = torch.randn(c, kv, d, generator=g, device="cuda").bfloat16()
    for f, t in ((edit, table), (edit_prefix, ptable)):
        if f is not None:
            f(t)
    q = (torch.randn(rows, heads, d, generator=g, device="cuda") * spread).bfloat16()
    sizes = [n] if sizes is None else sizes
    goff = np.cumsum([0] + list(sizes))
    kw = {}
    if len(prefix):
        kw = dict(prefix_table=ints(ptable), prefix_lengths=ints(list(prefix)))
        if not equal_groups:
            kw["group_offsets"] = ints(goff)
    row_off = None if rows_of is None and not first_row and not last_rows else ints(off)
    args = (q, k_pages, v_pages, ints(table), ints(lengths))
    out = ops.prefix_attention(*args, row_offsets=row_off, scale=scale, **kw)
    again = ops.prefix_attention(*args, row_offsets=row_off, scale=scale, **kw)
    torch.cuda.synchronize()
    want, width = P.prefix_attention_ref(f64(q), f64(k_pages), f64(v_pages), table, np.array(lengths), ptable if len(prefix) else None,
                                         list(prefix), None if row_off is None else off, goff, scale)
    got = f64(out)
    assert np.isfinite(got).all()
    err = np.abs(got - want) - (2.0 ** -8 * (np.abs(want) + width) + 2.0 ** -13 * width)
    assert (err <= 0).all(), f"largest excess {err.max():.3g} at {np.unravel_index(err.argmax(), err.shape)}, |want| up to {np.abs(want).max():.3g}"
    assert torch.equal(out.view(torch.int16), again.view(torch.int16)), "two calls differ"
    return out


HEADS = [(8, 8, 64), (32, 8, 128), (10, 2, 64), (12, 4, 128), (20, 1, 128), (4, 4, 128), (16, 1, 64)]


@pytest.mark.parametrize("heads,kv,d", HEADS)
@pytest.mark.parametrize("ps", [16, 24])
def test_attention_single_tokens_over_a_shared_prefix(ops, heads, kv, d, ps):
    check_attention(ops, lengths=[0, 1, 5, 17, 63, 64, 65, 130], prefix=[375], heads=heads, kv=kv, d=d, ps=ps)


@pytest.mark.parametrize("heads,kv,d", HEADS)
def test_attention_without_a_prefix(ops, heads, kv, d):
    check_attention(ops, lengths=[0, 3, 15, 16, 127, 128, 400], heads=heads, kv=kv, d=d)


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 63, 64, 127, 128, 129, 255, 257, 1000, 4100])
@pytest.mark.parametrize("heads,kv,d", [(8, 8, 64), (8, 2, 128)])
def test_attention_prefix_lengths(ops, prefix, heads, kv, d):
    check_attention(ops, lengths=[2, 0, 9], prefix=[prefix], heads=heads, kv=kv, d=d, seed=prefix)


@pytest.mark.parametrize("n", [1, 3, 16, 17, 40, 70, 140, 300])
@pytest.mark.parametrize("heads,kv,d", [(2, 2, 64), (4, 1, 128)])
def test_attention_numbers_of_sequences(ops, n, heads, kv, d):
    check_attention(ops, lengths=[(7 * i) % 40 for i in range(n)], prefix=[333], heads=heads, kv=kv, d=d, seed=n)


@pytest.mark.parametrize("heads,kv,d", [(2, 2, 64), (8, 2, 128), (5, 1, 128)])
@pytest.mark.parametrize("rows_of,lengths", [([5, 0, 1, 33], [0, 9, 31, 2]), ([130], [0]), ([1, 257], [70, 3]), ([64, 64], [0, 64]), ([300, 1, 2, 150], [0, 500, 0, 129])])
@pytest.mark.parametrize("prefix", [(), (200,)])
def test_attention_prompt_chunks(ops, heads, kv, d, rows_of, lengths, prefix):
    check_attention(ops, lengths=lengths, rows_of=rows_of, prefix=prefix, heads=heads, kv=kv, d=d, first_row=2, last_rows=3)


@pytest.mark.parametrize("heads,kv,d", [(4, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("tokens", [1, 20])
def test_attention_groups_of_different_sizes(ops, heads, kv, d, tokens):
    sizes = [3, 0, 1, 12, 5]
    n = sum(sizes)
    check_attention(ops, lengths=[(11 * i) % 30 - (i % 7 == 3) * 100 for i in range(n)], rows_of=None if tokens == 1 else [(5 * i) % tokens for i in range(n)],
                    prefix=[100, 40, 0, 700, 1], sizes=sizes, heads=heads, kv=kv, d=d)


def test_attention_equal_groups_and_sequences_of_no_group(ops):
    check_attention(ops, lengths=[1, 2, 3, 4, 5, 6], prefix=[50, 130, 20], sizes=[2, 2, 2], equal_groups=True)
    check_attention(ops, lengths=[1, 2, 3, 4, 5, 6], prefix=[50, 130], sizes=[2, 2])  # the last two share nothing


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("heads,kv,d", [(4, 4, 64), (8, 2, 128)])
def test_attention_dropped_pages_and_empty_rows(ops, heads, kv, d, tokens):
    """Pages missing at the start, in the middle, all of them: rows with no key at all are zero."""
    def edit(t):
        t[0, 0] = -1
        t[1, 1:3] = [-1, 10 ** 6]
        t[2, :] = -7

    def edit_prefix(t):
        t[0, 3:9] = -1
        t[1, :] = 2 ** 31 - 1

    n = [40, 70, 90, 5]
    out = check_attention(ops, lengths=n, rows_of=None if tokens == 1 else [tokens] * 4, prefix=[333, 200, 0], sizes=[2, 1, 1], heads=heads, kv=kv, d=d, edit=edit, edit_prefix=edit_prefix)
    assert not f64(out[2 * tokens:3 * tokens]).any()


@pytest.mark.parametrize("spread", [0.0, 6.0])
@pytest.mark.parametrize("heads,kv,d,n", [(4, 4, 64, 5), (8, 2, 128, 40)])
def test_attention_flat_and_peaked_rows(ops, spread, heads, kv, d, n):
    check_attention(ops, lengths=[60 + i for i in range(n)], prefix=[900], heads=heads, kv=kv, d=d, spread=spread, scale=None if spread else 1.0)


@pytest.mark.parametrize("layout", ["heads", "wide"])
@pytest.mark.parametrize("tokens", [1, 50])
def test_attention_layouts_of_the_cache(ops, layout, tokens):
    check_attention(ops, lengths=[20, 3, 47], rows_of=[tokens] * 3, prefix=[150], layout=layout)


@pytest.mark.parametrize("ps", [1, 7, 100, 128, 512])
@pytest.mark.parametrize("tokens", [1, 90])
def test_attention_page_sizes(ops, ps, tokens):
    check_attention(ops, lengths=[20, 3, 147], rows_of=[tokens] * 3, prefix=[260], ps=ps, kv=2, heads=2)


def test_attention_tables_wider_than_the_lengths(ops):
    """A table sized for the longest sequence that may come: most of it unused."""
    check_attention(ops, lengths=[20, 3, 0], prefix=[260], extra_width=5000)
    check_attention(ops, lengths=[20, 3, 0], rows_of=[80, 1, 30], prefix=[260], extra_width=5000, kv=2, heads=8, d=128)


@pytest.mark.parametrize("heads,kv,d", [(2, 2, 64), (4, 1, 128)])
def test_attention_long_own_context(ops, heads, kv, d):
    check_attention(ops, lengths=[9000, 17, 2500], heads=heads, kv=kv, d=d, ps=64)
    check_attention(ops, lengths=[3000, 17], rows_of=[35, 70], heads=heads, kv=kv, d=d, ps=64)


def dense_reference(q, k_pages, v_pages, table, length, ptable, prefix, groups, scale=None):
    """fp64 on the device, for sequences of one length and groups of one size: q [n, tokens, heads, d], `length` own tokens before them.
    Returns (out, spread) like the oracle."""
    n, tokens, heads, d = q.shape
    ps, kv = k_pages.shape[1], k_pages.shape[2]
    own = length + tokens
    out, spread = torch.empty(n, tokens, heads, d, dtype=torch.float64, device="cuda"), torch.empty(n, tokens, heads, d, dtype=torch.float64, device="cuda")
    j = torch.arange(own, device="cuda")
    late = j > length + torch.arange(tokens, device="cuda")[:, None]
    jp = torch.arange(prefix, device="cuda")
    for s in range(n):
        parts = []
        for cache in (k_pages, v_pages):
            x = cache[table[s].long()[j // ps], j % ps]
            if prefix:
                x = torch.cat([cache[ptable[s // (n // groups)].long()[jp // ps], jp % ps], x])
            parts.append(x.double().permute(1, 0, 2))  # [kv, keys, d]
        x = torch.einsum("htd,hjd->htj", q[s].double().transpose(0, 1), parts[0].repeat_interleave(heads // kv, 0)) * (d ** -0.5 if scale is None else scale)
        x[:, :, prefix:].masked_fill_(late, float("-inf"))
        w = torch.softmax(x, -1)
        v = parts[1].repeat_interleave(heads // kv, 0)
        out[s], spread[s] = (w @ v).transpose(0, 1), (w @ v.abs()).transpose(0, 1)
    return out, spread


@pytest.mark.parametrize("n,tokens,groups,heads,kv,d,length,prefix", [
    (1250, 3, 50, 64, 8, 128, 150, 300),   # more items for every stream of the tile kernel than are looked up at a time, pairs for the prefixes
    (50, 600, 5, 32, 32, 64, 3, 100),      # the same for pairs that take prefix and own tokens in a row
    (600, 1, 3, 16, 4, 64, 300, 5000),     # many rows of a group, few of a sequence
    (3000, 1, 1, 8, 8, 64, 20, 0),         # short own runs, a warp each
    (2, 1, 2, 32, 8, 128, 40000, 30000),   # few rows over many keys: many parts of a row
    (7, 700, 1, 12, 4, 128, 900, 3000),
    (1500, 40, 1, 2, 2, 64, 290, 50),      # more owners than a warp counts at a time, with own tiles
    (1100, 140, 11, 2, 1, 64, 0, 40),      # the same for pairs
])
def test_attention_large_calls(ops, n, tokens, groups, heads, kv, d, length, prefix):
    ps = 16
    width, pw = -(-(length + tokens) // ps), -(-prefix // ps)
    g = torch.Generator(device="cuda").manual_seed(n)
    order = torch.randperm(n * width + groups * pw, generator=g, device="cuda").to(torch.int32)
    table, ptable = order[:n * width].view(n, width), order[n * width:].view(groups, pw)
    k_pages, v_pages = make_cache(order.numel(), ps, kv, d, seed=n)
    q = torch.randn(n, tokens, heads, d, generator=g, device="cuda").bfloat16()
    kw = dict(prefix_table=ptable, prefix_lengths=ints([prefix] * groups)) if prefix else {}
    off = None if tokens == 1 else ints([tokens * i for i in range(n + 1)])
    out = ops.prefix_attention(q.view(-1, heads, d), k_pages, v_pages, table, ints([length] * n), row_offsets=off, **kw).view(q.shape)
    want, spread = dense_reference(q, k_pages, v_pages, table, length, ptable, prefix, groups)
    err = (out.double() - want).abs() - (2.0 ** -8 * (want.abs() + spread) + 2.0 ** -13 * spread)
    assert (err <= 0).all(), err.max().item()


@pytest.mark.parametrize("length", [1600, 3600])
def test_attention_many_prompts_with_odd_ends(ops, length):
    """Runs whose last rows leave the second tile of a pair without any, several of them per SM, over more keys than there are masks kept; rows
    that a single key rules."""
    n, tokens, heads, d, ps, prefix = 80, 300, 4, 64, 16, 137
    width, pw = -(-(length + tokens) // ps), -(-prefix // ps)
    order = torch.randperm(n * width + pw, generator=torch.Generator().manual_seed(1)).to("cuda", torch.int32)
    table, ptable = order[:n * width].view(n, width), order[n * width:].view(1, pw)
    k_pages, v_pages = make_cache(order.numel(), ps, heads, d)
    q = (torch.randn(n, tokens, heads, d, generator=torch.Generator().manual_seed(2)) * 6).to("cuda", torch.bfloat16)
    out = ops.prefix_attention(q.view(-1, heads, d), k_pages, v_pages, table, ints([length] * n), ptable, ints([prefix]),
                               row_offsets=ints([tokens * i for i in range(n + 1)])).view(q.shape)
    want, spread = dense_reference(q, k_pages, v_pages, table, length, ptable, prefix, 1)
    err = (out.double() - want).abs() - (2.0 ** -8 * (want.abs() + spread) + 2.0 ** -13 * spread)
    assert (err <= 0).all(), err.max().item()


@pytest.mark.parametrize("seed", range(40))
def test_attention_random_calls(ops, seed):
    rng = np.random.default_rng(seed)
    heads, kv, d = [(2, 2, 64), (8, 2, 64), (6, 1, 128), (4, 4, 128), (10, 2, 128), (16, 1, 64)][rng.integers(6)]
    groups = int(rng.integers(0, 5))
    sizes = [int(rng.integers(0, 9)) for _ in range(groups)] if groups else [int(rng.integers(1, 12))]
    n = max(sum(sizes) + int(rng.integers(0, 2)), 1)  # perhaps a sequence of no group
    tokens = [int(rng.integers(0, [2, 9, 40, 130][rng.integers(4)])) for _ in range(n)] if rng.random() < 0.7 else None
    top = [3, 60, 300][rng.integers(3)]
    lengths = [int(rng.integers(-1, top)) for _ in range(n)]
    prefix = [int(rng.integers(0, [5, 200, 900][rng.integers(3)])) for _ in range(groups)]

    def edit(t):
        if rng.random() < 0.5:
            t[rng.random(t.shape) < 0.2] = [-1, 10 ** 7][rng.integers(2)]

    check_attention(ops, lengths=lengths, rows_of=tokens, prefix=prefix, sizes=sizes if groups else None, heads=heads, kv=kv, d=d,
                    ps=[1, 5, 16, 24, 32, 64][rng.integers(6)], layout=["tokens", "heads", "wide"][rng.integers(3)], spread=[0.5, 1.0, 4.0][rng.integers(3)],
                    seed=seed, edit=edit, edit_prefix=edit, first_row=int(rng.integers(0, 3)) if tokens else 0, last_rows=int(rng.integers(0, 3)) if tokens else 0,
                    extra_width=[0, 0, 3, 400][rng.integers(4)])


def test_attention_offsets_beyond_32_bits(ops):
    """Pages more than 2^31 elements into the cache."""
    ps, kv, d = 64, 8, 128
    pages = 2 ** 31 // (ps * kv * d) + 40
    k_pages = torch.empty(pages, ps, kv, d, dtype=torch.bfloat16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    rng = np.random.default_rng(0)
    high = rng.permutation(np.arange(pages - 30, pages))
    small = [torch.randn(30, ps, kv, d, device="cuda").bfloat16() for _ in range(2)]
    table, ptable = np.arange(6).reshape(2, 3), np.arange(6, 16)[None]
    lengths, rows_of = [130, 0], [3, 61]
    q = torch.randn(64, 32, d, device="cuda").bfloat16()
    kv_new = [torch.randn(64, kv, d, device="cuda").bfloat16() for _ in range(2)]
    results = []
    for k, v, ids in ((small[0].clone(), small[1].clone(), np.arange(30)), (k_pages, v_pages, high)):
        ids_t = torch.from_numpy(ids).cuda()
        if k is k_pages:
            k[ids_t], v[ids_t] = small[0], small[1]
        t, pt, off = ints(ids[table]), ints(ids[ptable]), ints([0, 3, 64])
        qr = ops.kv_append(*kv_new, k, v, t, ints(lengths), q=q, row_offsets=off, rotary=ops.rotary_table(200, d))
        out = ops.prefix_attention(qr, k, v, t, ints(lengths), pt, ints([600]), row_offsets=off)
        one = ops.prefix_attention(qr[:2], k, v, t, ints([132, 0]), pt, ints([600]))
        results.append((qr, out, one, k[ids_t]))
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_attention_nan_and_infinities_in_seen_places_stay_with_their_rows(ops):
    """A NaN among the keys of one sequence reaches that sequence only."""
    k_pages, v_pages = make_cache(8, 16, 2, 64)
    t = ints([[0], [1], [2]])
    q = torch.randn(3, 2, 64, device="cuda").bfloat16()
    want = ops.prefix_attention(q, k_pages, v_pages, t, ints([9, 9, 9]), ints([[3, 4]]), ints([25]))
    k_pages[1, 4, 0, 3] = float("nan")
    v_pages[2, 2, 1, 5] = float("inf")
    got = ops.prefix_attention(q, k_pages, v_pages, t, ints([9, 9, 9]), ints([[3, 4]]), ints([25]))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, 1], want[1, 1]) and torch.equal(got[2, 0], want[2, 0])
    assert torch.isnan(got[1, 0]).all() and torch.isinf(got[2, 1, 5])
    keep = torch.arange(64, device="cuda") != 5
    assert torch.equal(got[2, 1][keep], want[2, 1][keep])


@pytest.mark.parametrize("heads,kv,d,tokens,length,prefix", [
    (4, 4, 64, 3, 37, 90), (4, 2, 64, 7, 0, 0), (8, 8, 128, 5, 61, 0), (8, 2, 128, 4, 14, 200),     # few rows
    (4, 4, 64, 40, 250, 90), (8, 2, 128, 30, 170, 0), (8, 1, 128, 12, 300, 20),                       # more
    (4, 4, 64, 300, 70, 200), (8, 2, 128, 300, 0, 0), (2, 1, 128, 130, 5, 130)])                      # prompts
def test_attention_values_that_are_not_finite_stay_out_of_earlier_rows(ops, heads, kv, d, tokens, length, prefix):
    """Infinities and NaN among the new tokens: the rows in front of them do not see them."""
    ps, n = 16, 3
    own, pre = -(-(length + tokens) // ps), -(-prefix // ps)
    table = np.arange(n * own).reshape(n, own)
    ptable = n * own + np.arange(pre)[None]
    k_pages, v_pages = make_cache(n * own + pre + 1, ps, kv, d)
    at = lambda s, i: (int(table[s, (length + i) // ps]), (length + i) % ps)  # noqa: E731
    for i in {tokens // 2, tokens - 1}:
        v_pages[at(0, i)][0, 5] = float("inf")
        v_pages[at(0, i)][kv - 1, d - 1] = float("nan")
    for i in range(tokens - tokens // 3, tokens):  # many of them, in tiles that follow one another
        v_pages[at(1, i)][:, i % d] = float("-inf") if i % 2 else float("nan")
    k_pages[at(1, tokens - 1)][kv - 1, 3] = float("nan")
    q = torch.randn(n * tokens, heads, d, device="cuda").bfloat16()
    off = np.arange(n + 1) * tokens
    kw = dict(prefix_table=ints(ptable), prefix_lengths=ints([prefix])) if prefix else {}
    got = f64(ops.prefix_attention(q, k_pages, v_pages, ints(table), ints([length] * n), row_offsets=ints(off), **kw))
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        want, width = P.prefix_attention_ref(f64(q), f64(k_pages), f64(v_pages), table, np.array([length] * n), ptable if prefix else None, [prefix], off)
    ok = np.isfinite(want)
    assert ok[0].all() and ok[tokens // 2 - 1].all() and not ok[tokens - 1].all() and ok[2 * tokens:].all()
    assert (np.isfinite(got) == ok).all(), f"{(np.isfinite(got) != ok).sum()} values"
    assert (np.isnan(got) == np.isnan(want)).all() and (got[np.isinf(want)] == want[np.isinf(want)]).all()
    assert (np.abs(got - want)[ok] <= (2.0 ** -8 * (np.abs(want) + width) + 2.0 ** -13 * width)[ok]).all()


def test_attention_nothing(ops):
    k_pages, v_pages = make_cache(2, 16, 2, 64)
    e = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    assert ops.prefix_attention(e, k_pages, v_pages, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([])).shape == (0, 2, 64)
    q = torch.ones(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = ops.prefix_attention(q, k_pages, v_pages, torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([]), row_offsets=ints([0]))
    assert not out.any()
    none = torch.empty(0, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = ops.prefix_attention(q, none, none, torch.full((4, 2), 0, dtype=torch.int32, device="cuda"), ints([3] * 4),
                               torch.zeros(1, 0, dtype=torch.int32, device="cuda"), ints([9]))
    assert not out.any()


def test_attention_garbage_in_the_tables_stays_inside_the_cache(ops):
    """Lengths, offsets and group offsets that make no sense: finite or zero results, no fault."""
    k_pages, v_pages = make_cache(6, 16, 2, 64)
    q = torch.randn(40, 2, 64, device="cuda").bfloat16()
    big = 2 ** 31 - 1
    for off in ([0, 20, 40], [40, 20, 0], [-big, big, 3], [5, 5, big], [big, big, big]):
        for go in ([0, 1, 2], [big, -4, 1], [-big, big, big], [2, 1, 0]):
            out = ops.prefix_attention(q, k_pages, v_pages, ints([[0, 1], [2, big]]), ints([big, 7]), ints([[3, -big], [4, 5]]), ints([big, -3]),
                                       row_offsets=ints(off), group_offsets=ints(go))
            torch.cuda.synchronize()
            assert torch.isfinite(out.float()).all()


def test_attention_views_strides_and_out(ops):
    k_pages, v_pages = make_cache(8, 16, 2, 64)
    wide = torch.randn(5, 6 * 64 + 8, device="cuda").bfloat16()
    q = wide[:, 8:].unflatten(1, (6, 64))[:, 1:5]
    t, n = ints([[0], [1], [2], [3], [4]]), ints([3, 9, 15, 0, -1])
    want = ops.prefix_attention(q.contiguous(), k_pages, v_pages, t, n, ints([[5, 6]]), ints([30]))
    assert torch.equal(ops.prefix_attention(q, k_pages, v_pages, t, n, ints([[5, 6]]), ints([30])), want)
    odd = torch.empty(5 * 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(5, 4, 64).copy_(q)  # 2-byte aligned
    assert torch.equal(ops.prefix_attention(odd, k_pages, v_pages, t, n, ints([[5, 6]]), ints([30])), want)
    out = torch.full((5, 4, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    got = ops.prefix_attention(q, k_pages, v_pages, t, n, ints([[5, 6]]), ints([30]), out=out[:, :, 1])
    assert torch.equal(got, want) and (out[:, :, 0] == 7).all()
    strided = ints([[0, 9], [1, 9], [2, 9], [3, 9], [4, 9]])
    assert torch.equal(ops.prefix_attention(q, k_pages, v_pages, strided[:, ::2], n, ints([[5, 6]]), ints([30])), want)


# ------------------------------------------------------------------------------------------------ together


def _decode(ops, steps, heads, kv, d, n, prefix, seed=0, tokens=1):
    """`steps` steps of append + attend; returns the results and what a cache that is not paged gives."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps = 16
    width = -(-steps * tokens // ps)
    pw = -(-prefix // ps)
    pages = n * width + pw
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    t, pt = order[:n * width].view(n, width), order[n * width:].view(1, pw)
    k_pages, v_pages = make_cache(pages, ps, kv, d, fill=float("nan"))
    rot = ops.rotary_table(prefix + steps * tokens, d)
    pk, pv = (torch.randn(prefix, kv, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    ops.kv_append(pk, pv, k_pages, v_pages, pt, ints([0]), rotary=rot, row_offsets=ints([0, prefix]))
    lengths, starts, plen = ints([0] * n), ints([prefix] * n), ints([prefix])
    off = None if tokens == 1 else ints([tokens * i for i in range(n + 1)])
    results = []
    for _ in range(steps):
        x = torch.randn(n * tokens, (heads + 2 * kv) * d, generator=g, device="cuda").bfloat16()
        q, k, v = x.split([heads * d, kv * d, kv * d], dim=1)
        qr = ops.kv_append(k.unflatten(1, (kv, d)), v.unflatten(1, (kv, d)), k_pages, v_pages, t, lengths, q=q.unflatten(1, (heads, d)), rotary=rot,
                           row_offsets=off, starts=starts)
        results.append((qr, ops.prefix_attention(qr, k_pages, v_pages, t, lengths, pt, plen, row_offsets=off)))
        lengths = lengths + tokens
    return results, (k_pages, v_pages, t, pt)


@pytest.mark.parametrize("heads,kv,d,n,tokens", [(8, 8, 64, 10, 1), (8, 2, 128, 33, 1), (4, 4, 64, 3, 30)])
def test_steps_of_decoding(ops, heads, kv, d, n, tokens):
    steps, prefix = 6, 210
    results, (k_pages, v_pages, t, pt) = _decode(ops, steps, heads, kv, d, n, prefix, tokens=tokens)
    torch.cuda.synchronize()
    off = np.arange(n + 1) * tokens
    for step, (q, out) in enumerate(results):
        want, width = P.prefix_attention_ref(f64(q), np.nan_to_num(f64(k_pages)), np.nan_to_num(f64(v_pages)), f64(t).astype(int), np.array([step * tokens] * n),
                                             f64(pt).astype(int), [prefix], off, [0, n])
        assert (np.abs(f64(out) - want) <= 2.0 ** -8 * (np.abs(want) + width) + 2.0 ** -13 * width).all(), step


def test_a_step_right_behind_the_one_that_wrote_its_keys(ops):
    """Append and attention overlap with what is in front of them; many steps in a row give the same bits each time."""
    first, _ = _decode(ops, 40, 8, 8, 64, 10, 375)
    for _ in range(5):
        again, _ = _decode(ops, 40, 8, 8, 64, 10, 375)
        assert all(torch.equal(a[1], b[1]) for a, b in zip(first, again))


def test_other_streams_and_graphs(ops):
    want, _ = _decode(ops, 3, 8, 2, 128, 20, 300)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = _decode(ops, 3, 8, 2, 128, 20, 300)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a[1], b[1]) for a, b in zip(want, got))
    # a captured step follows lengths that are moved on the device
    ps, kv, d, n = 16, 2, 64, 6
    k_pages, v_pages = make_cache(40, ps, kv, d)
    t, pt = ints(np.arange(24).reshape(6, 4)), ints([[30, 31, 32]])
    lengths, plen, starts = ints([0, 3, 9, 15, 16, 31]), ints([40]), ints([40] * 6)
    rot = ops.rotary_table(200, d)
    x = torch.randn(n, 8, d, device="cuda").bfloat16()
    state = k_pages.clone(), v_pages.clone(), lengths.clone()

    def step():
        q = ops.kv_append(x[:, 4:6], x[:, 6:], k_pages, v_pages, t, lengths, q=x[:, :4], rotary=rot, starts=starts)
        out = ops.prefix_attention(q, k_pages, v_pages, t, lengths, pt, plen)
        lengths.add_(1)
        return out

    eager = [step().clone() for _ in range(4)]
    for a, b in zip((k_pages, v_pages, lengths), state):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for want in eager:
        graph.replay()
        assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------ refusals


def test_refusals(ops):
    k_pages, v_pages = make_cache(4, 16, 2, 64)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    t, n = ints([[0], [1], [2]]), ints([0, 0, 0])
    ok = dict(k=k, v=k, k_pages=k_pages, v_pages=v_pages, page_table=t, lengths=n)

    def append(**kw):
        a = {**ok, **kw}
        return ops.kv_append(a.pop("k"), a.pop("v"), a.pop("k_pages"), a.pop("v_pages"), a.pop("page_table"), a.pop("lengths"), **a)

    append()
    for err, kw in [
        (RuntimeError, dict(k=k.cpu())), (RuntimeError, dict(lengths=n.cpu())), (RuntimeError, dict(k_pages=k_pages.cpu(), v_pages=v_pages.cpu())),
        (ValueError, dict(v=k[:2])), (ValueError, dict(k=k[:, :1])), (ValueError, dict(k=k[0])), (TypeError, dict(v=k.float())), (TypeError, dict(k=k.half(), v=k.half())),
        (ValueError, dict(k_pages=k_pages.float(), v_pages=v_pages.float())), (ValueError, dict(v_pages=v_pages[:3])), (ValueError, dict(k_pages=k_pages[..., ::2], v_pages=v_pages[..., ::2], k=k[..., ::2], v=k[..., ::2])),
        (ValueError, dict(page_table=t.long())), (ValueError, dict(page_table=t[0])), (ValueError, dict(lengths=n[:2])), (ValueError, dict(lengths=n.long())),
        (ValueError, dict(page_table=t[:2], lengths=n[:2])), (ValueError, dict(row_offsets=ints([0, 1, 2]))), (ValueError, dict(starts=ints([0]))),
        (ValueError, dict(q_out=q)), (ValueError, dict(q=q[:2])), (TypeError, dict(q=q.float())), (ValueError, dict(q=q, q_out=q.float())), (ValueError, dict(q=q, q_out=q[:, :3])),
        (ValueError, dict(rotary=torch.zeros(9, 40, device="cuda"))), (ValueError, dict(rotary=torch.zeros(9, 128, device="cuda"))), (ValueError, dict(rotary=torch.zeros(9, 64, device="cuda", dtype=torch.bfloat16))),
        (ops._lib.VeloxError, dict(k_pages=k_pages[:1].expand(4, 16, 2, 64))),
    ]:
        with pytest.raises(err):
            append(**kw)
    p, m = ints([[3]]), ints([9])

    def attend(*a, **kw):
        return ops.prefix_attention(*a, **kw)

    attend(q, k_pages, v_pages, t, n, p, m)
    odd = [make_cache(4, 16, 2, 96)[0]] * 2
    for err, a, kw in [
        (RuntimeError, (q.cpu(), k_pages, v_pages, t, n), {}), (TypeError, (q.float(), k_pages, v_pages, t, n), {}), (ValueError, (q[:, :3], k_pages, v_pages, t, n), {}),
        (ValueError, (q[:2], k_pages, v_pages, t, n), {}), (ValueError, (q[..., :32], k_pages, v_pages, t, n), {}), (ValueError, (q, k_pages, v_pages, t, n, p), {}),
        (ValueError, (q, k_pages, v_pages, t, n, None, m), {}), (ValueError, (q, k_pages, v_pages, t, n, ints([[1], [2]]), ints([3, 4])), {}),
        (ValueError, (q, k_pages, v_pages, t, n, p, m), dict(group_offsets=ints([0, 1, 3]))), (ValueError, (q, k_pages, v_pages, t, n, p.long(), m), {}),
        (ValueError, (q, k_pages, v_pages, t, n), dict(row_offsets=ints([0, 3]))), (ValueError, (q, k_pages, v_pages, t, n), dict(out=q.float())),
        (ValueError, (q, k_pages, v_pages, t, n), dict(out=q[:2])), (ValueError, (torch.zeros(3, 4, 96, device="cuda", dtype=torch.bfloat16), *odd, t, n), {}),
    ]:
        with pytest.raises(err):
            attend(*a, **kw)
    assert ops._lib.device_status() == 0


def test_native_and_general_routes_agree(ops, monkeypatch):
    """The native host path and the Python code behind it pass the same descriptors on."""
    class Declines:
        @staticmethod
        def kv_append(*a):
            return None

        prefix_attention = kv_append

        @staticmethod
        def launches():
            return 0

    def results():
        out = []
        for kw in (dict(heads=8, kv=8, d=64, n=10), dict(heads=8, kv=2, d=128, n=5, tokens=20)):
            out += [t for pair in _decode(ops, 3, prefix=100, **kw)[0] for t in pair]
        k_pages, v_pages = make_cache(6, 16, 2, 64, "heads")
        x = torch.randn(4, 3, 2, 64, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
        rot = ops.rotary_table(99, 32)
        q_out = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
        t, n, off = ints([[0, 1, 2], [3, 4, 5]]), ints([5, 17]), ints([0, 3, 4])
        got = ops.kv_append(x[:, 0], x[:, 1], k_pages, v_pages, t, n, q=x[:, 2], rotary=rot, interleaved=True, row_offsets=off, starts=ints([9, 1]), q_out=q_out)
        assert got is q_out and ops.kv_append(x[:, 0], x[:, 1], k_pages, v_pages, t, n, row_offsets=off) is None
        o = torch.zeros_like(q_out)
        assert ops.prefix_attention(q_out, k_pages, v_pages, t, n, ints([[0], [3]]), ints([9, 16]), row_offsets=off, group_offsets=ints([0, 1, 2]), scale=0.3, out=o) is o
        return out + [q_out, o, k_pages, v_pages]

    before = ops.launch_count()
    first = results()
    assert ops.launch_count() > before
    assert ops._native is not None
    monkeypatch.setattr(ops, "_native", Declines)
    second = results()
    for a, b in zip(first, second):
        assert torch.equal(a, b)
