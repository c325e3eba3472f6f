"""kv_append, kv_values and prefix_attention on a cache in 4 bits, against their definitions (oracle/paged.py).

What kv_append stores is defined to the bit: bytes are compared.  Attention, tolerances by the number formats: a probability is rounded to fp16
(2^-11 of it, so 2^-11 sum_j w_j |v_j| of a result; below 2^-14 of the largest by 2^-25 of the row's largest, at most 2^-25 n over n keys), the result once
to bf16 (2^-8); a query's values below 2^-17 of its row's largest by 2^-25 of that, fp32 products, sums and exponentials: a weight changes by less than 2^-13 at
the scores used here (|s| < 60)."""

import numpy as np
import pytest
import torch

from oracle import paged as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from velox_voice_b200 import ops as o

    return o


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def host(t):
    return t.detach().cpu().numpy()


def pages_of(total, ps, kv, d, seed=0, low=0x18, high=0x31):
    """random codes, scales between 1/16 and 1/2"""
    g = np.random.default_rng(seed)
    x = g.integers(0, 256, (total, kv, ps // 16, 9 * d), dtype=np.uint8)
    x[..., 8 * d:] = g.integers(low, high, x[..., 8 * d:].shape, dtype=np.uint8)
    return x


def tables(counts, total, seed=0, width=None):
    order = np.random.default_rng(seed).permutation(total)
    t = np.full((len(counts), max(max(counts), 1) if width is None else width), -1, dtype=np.int64)
    at = 0
    for i, c in enumerate(counts):
        t[i, :c] = order[at:at + c]
        at += c
    assert at <= total
    return t, order[at:]


# ------------------------------------------------------------------------------------------------ kv_append


def check_append(ops, *, rows_of, lengths, heads=4, kv=2, d=64, ps=16, rot=64, dtype=torch.bfloat16, interleaved=False, starts=None, positions=None,
                 edit_table=None, offsets=True, first_row=0, last_rows=0, shift=0, seed=0, k_scale=1.0, v_scale=1.0, edit=None, with_q=True, apart=False):
    n = len(lengths)
    rows = first_row + sum(rows_of) + last_rows
    off = np.cumsum([first_row] + list(rows_of))
    counts = [-(-(max(l, 0) + c) // ps) for l, c in zip(lengths, rows_of)]
    total = sum(counts) + 2
    table, _ = tables(counts, total, seed)
    if edit_table is not None:
        edit_table(table)
    before = [pages_of(total, ps, kv, d, seed + i) for i in range(2)]
    k_pages, v_pages = (torch.from_numpy(b).cuda() for b in before)
    if apart:  # pages of a larger pool, one behind the other with a gap
        k_pages, v_pages = (torch.stack([x, x], 1)[:, 0] for x in (k_pages, v_pages))
        assert not k_pages.is_contiguous()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, (heads + 2 * kv) * d + shift, generator=g, device="cuda")
    if edit is not None:
        edit(x)
    x = x.to(dtype)[:, shift:]
    q, k, v = x[:, :heads * d].unflatten(1, (heads, d)), x[:, heads * d:(heads + kv) * d].unflatten(1, (kv, d)), x[:, (heads + kv) * d:].unflatten(1, (kv, d))
    start = [0] * n if starts is None else starts
    last = max([s + max(l, 0) + c for s, l, c in zip(start, lengths, rows_of)] + [1])
    rotary = ops.rotary_table(last if positions is None else positions, rot) if rot else None
    kw = dict(rotary=rotary, interleaved=interleaved, row_offsets=ints(off) if offsets else None, starts=None if starts is None else ints(starts))
    q_out = ops.kv_append(k, v, k_pages, v_pages, ints(table), ints(lengths), q=q if with_q else None, k_scale=k_scale, v_scale=v_scale, **kw)
    torch.cuda.synchronize()
    want = P.kv_append_fp4_ref(host(k.float()), host(v.float()), *before, table, np.array(lengths), None if rotary is None else host(rotary), interleaved,
                               off if offsets else None, starts, k_scale, v_scale)
    for got, w in zip((k_pages, v_pages), want):
        # (a value of -0 may have either sign)
        got = host(got)
        same = got == w
        if not same.all():
            a, b = P.fp4_values(got), P.fp4_values(w)
            assert (a == b).all(), f"{(a != b).sum()} values of {a.size} differ"
            assert (got[..., 8 * d:] == w[..., 8 * d:]).all()
    if with_q:  # as on a bf16 cache
        b16 = torch.zeros(total, ps, kv, d, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(q_out, ops.kv_append(k, v, b16, b16.clone(), ints(table), ints(lengths), q=q, **kw))
    else:
        assert q_out is None
    return k_pages, v_pages


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,d,rot,ps", [(8, 8, 64, 64, 16), (32, 8, 128, 128, 64), (6, 2, 128, 64, 48), (4, 1, 256, 16, 16), (3, 3, 16, 16, 16), (5, 5, 80, 48, 32),
                                               (4, 2, 64, 0, 16), (2, 2, 112, 96, 16)])
def test_append_single_tokens(ops, dtype, interleaved, heads, kv, d, rot, ps):
    check_append(ops, rows_of=[1] * 8, lengths=[0, 1, 15, 16, ps - 1, ps, 5 * ps + 3, 200], heads=heads, kv=kv, d=d, rot=rot, ps=ps, dtype=dtype, interleaved=interleaved, offsets=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 3])
def test_append_ragged_rows(ops, dtype, shift):
    check_append(ops, rows_of=[5, 0, 33, 1, 0, 200, 17], lengths=[0, 4, 15, 16, 9, 70, 1], dtype=dtype, starts=[0, 3, 375, 0, 1, 12, 9], seed=3, shift=shift, ps=32)


@pytest.mark.parametrize("rows", [1, 2, 700, 3001])
def test_append_one_long_sequence(ops, rows):
    check_append(ops, rows_of=[rows], lengths=[3], heads=2, kv=1, seed=rows, dtype=torch.float32)


def test_append_without_queries_and_into_pages_apart(ops):
    check_append(ops, rows_of=[40, 3], lengths=[1, 2], with_q=False, apart=True)


def test_append_leaves_out_what_has_no_place(ops):
    def edit(t):
        t[0, 1] = -1
        t[2, 0] = 10 ** 6
        t[3, :] = -(2 ** 31)

    check_append(ops, rows_of=[40, 9, 20, 5, 12], lengths=[0, -1, 3, 0, -2 ** 31], edit_table=edit, first_row=3, last_rows=6, seed=5)
    check_append(ops, rows_of=[10, 10, 10], lengths=[0, 0, 0], starts=[0, 25, -4], positions=30, seed=6)


@pytest.mark.parametrize("k_scale,v_scale", [(2.0 ** -9, 2.0 ** 7), (2.0 ** 32, 2.0 ** -32)])
def test_append_with_scales(ops, k_scale, v_scale):
    check_append(ops, rows_of=[40, 9], lengths=[0, 7], k_scale=k_scale, v_scale=v_scale, dtype=torch.float32, seed=9,
                 edit=lambda x: x.mul_(torch.cat([torch.full((4 * 64 + 2 * 64,), k_scale), torch.full((2 * 64,), v_scale)]).cuda()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_borders_and_sizes(ops, dtype):
    """Values on the borders between codes and next to them, blocks of zeros, blocks whose scale is subnormal, zero or at its end."""
    def edit(x):
        rows = x.shape[0]
        border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.0], device="cuda")
        size = torch.tensor([2.0 ** e * m for e in range(-12, 10) for m in (1, 1.125, 1.375, 1.5, 1.875)], device="cuda")
        v = border * size[torch.arange(rows, device="cuda") % size.numel(), None]
        x[:, -64:-48], x[:, -48:-32], x[:, -32:-16], x[:, -16:] = v, v * (1 + 2.0 ** -23), v * (1 - 2.0 ** -24), 0.0

    check_append(ops, rows_of=[220], lengths=[0], edit=edit, dtype=dtype, rot=0)


def test_what_is_not_finite_is_stored_as_finite(ops):
    ps, kv, d = 16, 1, 64
    k = torch.randn(3, kv, d, device="cuda")
    k[0, 0, 5], k[1, 0, 20], k[2, 0, 40] = float("inf"), float("nan"), float("-inf")
    kp, vp = ops.fp4_pages(1, ps, kv, d), ops.fp4_pages(1, ps, kv, d)
    ops.kv_append(k, k.clone(), kp, vp, ints([[0]]), ints([0]), row_offsets=ints([0, 3]))
    x = ops.kv_values(kp)
    assert torch.isfinite(x).all() and x[0, 0, 0, 5] == 2688 and x[0, 2, 0, 40] == -2688


# ------------------------------------------------------------------------------------------------ kv_values


@pytest.mark.parametrize("d,ps,kv,n,g", [(64, 16, 1, 1, 1.0), (128, 48, 3, 5, 2.0 ** -20), (16, 16, 2, 3, 2.0 ** 32), (256, 32, 1, 2, 0.5), (80, 16, 7, 4, 1.0), (64, 16, 8, 900, 1.0)])
def test_values_of_any_bytes(ops, d, ps, kv, n, g):
    x = np.random.default_rng(d).integers(0, 256, (n, kv, ps // 16, 9 * d), dtype=np.uint8)
    want = P.fp4_values(x, g)
    t = torch.from_numpy(x).cuda()
    for pages in (t, torch.stack([t, t], 1)[:, 1]):
        got = ops.kv_values(pages, g)
        assert got.dtype == torch.bfloat16 and (host(got.double()) == want).all()
    out = torch.empty_like(got)
    assert ops.kv_values(t, g, out=out) is out and torch.equal(out, got)


def test_values_of_no_pages(ops):
    assert ops.kv_values(ops.fp4_pages(0, 32, 2, 64)).shape == (0, 32, 2, 64)


# ------------------------------------------------------------------------------------------------ prefix_attention


def attend(ops, *, lengths, rows_of, heads, kv, d, ps, prefix=None, sizes=None, edit=None, seed=0, q_gain=1.0, offsets=True, scale=None, k_scale=1.0, v_scale=1.0,
           group_offsets=False, first_row=0, last_rows=0, any_bytes=False, edit_q=None, width=None, shift=0):
    """Runs and compares; returns the operator's arguments and result.  `sizes`: sequences per group."""
    n = len(lengths)
    own = [-(-(max(l, 0) + t) // ps) for l, t in zip(lengths, rows_of)]
    shared = [-(-p // ps) for p in prefix] if prefix else []
    total = sum(own) + sum(shared) + 2
    if shared:
        pt, rest = tables(shared, total, seed)
        order = rest
    else:
        pt, order = None, np.random.default_rng(seed).permutation(total)
    table = np.full((n, (width or 0) + max(max(own), 1)), -1, dtype=np.int64)
    at = 0
    for i, c in enumerate(own):
        table[i, :c] = order[at:at + c]
        at += c
    if edit is not None:
        edit(table, pt)
    kp, vp = (pages_of(total, ps, kv, d, seed + i, *((0, 256) if any_bytes else (0x18, 0x31))) for i in range(2))
    rows = first_row + sum(rows_of) + last_rows
    off = np.cumsum([first_row] + list(rows_of))
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(rows, heads * d + shift, generator=g, device="cuda") * q_gain)
    if edit_q is not None:
        edit_q(q)
    q = q.bfloat16()[:, shift:].unflatten(1, (heads, d))
    go = np.cumsum([0] + list(sizes)) if group_offsets else None
    kt, vt = torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda()
    args = (q, kt, vt, ints(table), ints(lengths))
    if shared:
        args += (ints(pt), ints(prefix))
    kw = dict(row_offsets=ints(off) if offsets else None, scale=scale, k_scale=k_scale, v_scale=v_scale)
    if go is not None:
        kw["group_offsets"] = ints(go)
    out = ops.prefix_attention(*args, **kw)
    torch.cuda.synchronize()
    from velox_voice_b200 import _lib

    assert _lib.device_status() == 0
    want, spread = P.prefix_attention_ref(host(q.double()), P.fp4_values(kp, k_scale), P.fp4_values(vp, v_scale), table, np.array(lengths), pt, None if not prefix else np.array(prefix),
                                          off if offsets else None, go, scale)
    keys = max([max(l, 0) + t for l, t in zip(lengths, rows_of)]) + (max(prefix) if prefix else 0)
    most = np.abs(P.fp4_values(vp, v_scale)).max()
    err = np.abs(host(out.double()) - want)
    bound = 2.0 ** -8 * (np.abs(want) + 2.0 ** -9 * spread) + (2.0 ** -11 + 2.0 ** -13) * spread + 2.0 ** -25 * keys * most
    assert (err <= bound).all(), f"worst {np.max(err / np.maximum(bound, 1e-30)):.3g} of the tolerance, at {np.unravel_index(np.argmax(err / np.maximum(bound, 1e-30)), err.shape)}"
    return args, kw, out


HEADS = [(8, 8, 64), (4, 1, 64), (32, 8, 128), (5, 1, 128)]


@pytest.mark.parametrize("heads,kv,d", HEADS)
@pytest.mark.parametrize("ps", [16, 48])
def test_single_tokens_without_a_prefix(ops, heads, kv, d, ps):
    attend(ops, lengths=[0, 1, 14, 15, 16, 63, 64, 65, -1, 300], rows_of=[1] * 10, heads=heads, kv=kv, d=d, ps=ps, offsets=False)


@pytest.mark.parametrize("heads,kv,d", HEADS)
@pytest.mark.parametrize("prefix", [[1, 17], [16, 0], [375, 900]])
def test_hypotheses_over_prefixes(ops, heads, kv, d, prefix):
    attend(ops, lengths=[0, 3, 40, -1, 7, 100], rows_of=[1] * 6, heads=heads, kv=kv, d=d, ps=16, prefix=prefix, offsets=False, seed=1)
    attend(ops, lengths=[0, 3, 40, -1, 7, 100], rows_of=[1] * 6, heads=heads, kv=kv, d=d, ps=32, prefix=prefix, sizes=[2, 4], group_offsets=True, seed=2)


@pytest.mark.parametrize("heads,kv,d", HEADS)
@pytest.mark.parametrize("rows_of,lengths", [([5, 5, 5, 5], [0, 20, 33, 64]), ([1, 0, 9, 16, 17], [5, 5, 0, 15, 16]), ([40, 33], [0, 90]), ([130, 1, 128, 129], [0, 700, 3, -1]), ([300, 257], [100, 0])])
def test_several_rows_of_a_sequence(ops, heads, kv, d, rows_of, lengths):
    attend(ops, lengths=lengths, rows_of=rows_of, heads=heads, kv=kv, d=d, ps=16, seed=3)
    attend(ops, lengths=lengths, rows_of=rows_of, heads=heads, kv=kv, d=d, ps=32, prefix=[200], seed=4, first_row=2, last_rows=3)


@pytest.mark.parametrize("heads,kv,d", [(8, 8, 64), (32, 8, 128)])
def test_many_hypotheses_of_one_prefix(ops, heads, kv, d):
    attend(ops, lengths=[3 * i % 70 for i in range(40)], rows_of=[1] * 40, heads=heads, kv=kv, d=d, ps=16, prefix=[3000], offsets=False, seed=5)


@pytest.mark.parametrize("d", [64, 128])
def test_pages_that_are_not_there(ops, d):
    def edit(table, pt):
        table[0, 1], table[1, :], table[2, 2:] = -1, -1, 10 ** 6
        pt[0, 0], pt[0, 3:20], pt[1, :] = -1, -(2 ** 31), -1

    attend(ops, lengths=[50, 40, 90, 30], rows_of=[3, 2, 1, 20], heads=4, kv=2, d=d, ps=16, prefix=[1000, 77], edit=edit, seed=6)


@pytest.mark.parametrize("d", [64, 128])
def test_any_bytes_are_finite_values(ops, d):
    """Scale bytes of 0x7f and with a sign too, in places that are read and in those that are not.  Scores are small: q is."""
    attend(ops, lengths=[50, 7, 0], rows_of=[3, 1, 20], heads=4, kv=2, d=d, ps=16, prefix=[300], any_bytes=True, q_gain=2.0 ** -9, seed=7)


def test_rows_that_see_nothing_are_zeros(ops):
    (q, *_), _, out = attend(ops, lengths=[-1, 4, -5], rows_of=[2, 2, 2], heads=4, kv=2, d=64, ps=16, first_row=3, last_rows=4, seed=8)
    assert not out[:3].any() and not out[3:5].any() and not out[7:].any() and out[5:7].all()


@pytest.mark.parametrize("k_scale,v_scale,gain", [(2.0 ** -12, 2.0 ** 9, 2.0 ** 12), (2.0 ** 20, 2.0 ** -30, 2.0 ** -20)])
def test_scales_of_the_cache(ops, k_scale, v_scale, gain):
    attend(ops, lengths=[50, 7, 0], rows_of=[3, 1, 20], heads=4, kv=2, d=128, ps=16, prefix=[300], k_scale=k_scale, v_scale=v_scale, q_gain=gain, seed=9)


def test_queries_of_all_sizes(ops):
    """Rows whose largest values are 2^60 apart, and rows of values 2^20 apart."""
    def edit_q(q):
        q *= torch.exp2(torch.linspace(-30, 2, q.shape[0], device=q.device).round())[:, None]
        q[:, ::7] *= 2.0 ** -20

    attend(ops, lengths=[100, 30], rows_of=[30, 33], heads=4, kv=2, d=64, ps=16, edit_q=edit_q, seed=10)


def test_large_scores(ops):
    """One key takes all of the weight: scores of 2^100 and more."""
    d = 64
    kp = pages_of(4, 16, 1, d, 3)
    vp = pages_of(4, 16, 1, d, 4)
    q = torch.randn(6, 2, d, device="cuda").bfloat16() * torch.tensor([2.0 ** e for e in (10, 30, 60, 90, 100, 110)], device="cuda").bfloat16()[:, None, None]
    out = ops.prefix_attention(q, torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), ints([[0, 1, 2, 3]] * 6), ints([60] * 6))
    k, v = P.fp4_values(kp).reshape(64, d)[:61], P.fp4_values(vp).reshape(64, d)[:61]
    for r in range(6):
        for h in range(2):
            x = k @ host(q[r, h].double()) / 8
            top = np.sort(x)
            if top[-1] - top[-2] > 2.0 ** -18 * np.abs(top[-1]) + 60:
                assert np.allclose(host(out[r, h].double()), v[x.argmax()], rtol=2.0 ** -7)


def test_two_calls_give_the_same_bits_and_strided_results(ops):
    args, kw, out = attend(ops, lengths=[50, 7, 0, 90], rows_of=[3, 1, 20, 150], heads=8, kv=2, d=128, ps=16, prefix=[3000], seed=11, shift=3)
    assert torch.equal(out, ops.prefix_attention(*args, **kw))
    wide = torch.full((out.shape[0], 8, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(ops.prefix_attention(*args, out=wide[..., 128:], **kw), out) and (wide[..., :128] == 7).all()


def test_no_rows_and_no_pages(ops):
    kp = ops.fp4_pages(0, 16, 2, 64)
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    assert not ops.prefix_attention(q, kp, kp, ints([[0]] * 3), ints([4] * 3)).any()
    assert ops.prefix_attention(q[:0], kp, kp, ints([[0]] * 3), ints([4] * 3), row_offsets=ints([0] * 4)).shape == (0, 4, 64)


@pytest.mark.parametrize("d", [64, 128])
def test_appended_then_read_on_a_side_stream_and_in_a_graph(ops, d):
    """append, attend, as a step uses them; replayed with other inputs, and beside another graph."""
    kv, heads, ps, n = 2, 4, 16, 5
    table = ints([[3 * i + j for j in range(3)] for i in range(n)])
    lengths, rotary = ints([0, 3, 15, 16, 30]), ops.rotary_table(64, d)
    x = torch.empty(n, heads + 2 * kv, d, device="cuda", dtype=torch.bfloat16)

    def call(kp, vp):
        q = ops.kv_append(x[:, heads:heads + kv], x[:, heads + kv:], kp, vp, table, lengths, q=x[:, :heads], rotary=rotary)
        return ops.prefix_attention(q, kp, vp, table, lengths)

    def fresh():
        return [torch.from_numpy(pages_of(15, ps, kv, d, i)).cuda() for i in range(2)]

    x.normal_()
    caches = [fresh() for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = call(*caches[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, call(*fresh()))
    graphs = []
    for c in caches:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(*c)
        graphs.append((g, out, c))
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        for (g, _, c) in graphs:
            for t, f in zip(c, fresh()):
                t.copy_(f)
            g.replay()
        want = call(*fresh())
        for _, out, _ in graphs:
            assert torch.equal(out, want)


def test_refusals(ops):
    kp, vp = ops.fp4_pages(4, 16, 2, 64), ops.fp4_pages(4, 16, 2, 64)
    k, q = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    t, n = ints([[0], [1]]), ints([0, 0])
    b16 = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(k_scale=3.0), dict(v_scale=0.0), dict(k_scale=float("nan"))):
        with pytest.raises(ValueError, match="power of two"):
            ops.kv_append(k, k, kp, vp, t, n, **bad)
        with pytest.raises(ValueError, match="power of two"):
            ops.prefix_attention(q, kp, vp, t, n, **bad)
    with pytest.raises(ValueError, match="4 bits"):
        ops.kv_append(k, k, b16, b16, t, n, k_scale=2.0)
    with pytest.raises(ValueError, match="4 bits"):
        ops.prefix_attention(q, b16, b16, t, n, v_scale=2.0)
    for a, b in ((kp, b16), (b16, vp), (kp, vp[:3]), (kp[..., :567], vp[..., :567]), (ops.fp4_pages(4, 32, 2, 64).transpose(1, 2),) * 2, (kp.flatten()[8:8 + 3 * 1152].view(3, 2, 1, 576), vp[:3])):
        with pytest.raises(ValueError):
            ops.kv_append(k, k, a, b, t, n)
        with pytest.raises(ValueError):
            ops.prefix_attention(q, a, b, t, n)
    wide = ops.fp4_pages(4, 16, 2, 80)
    with pytest.raises(ValueError, match="64 or 128"):
        ops.prefix_attention(torch.zeros(2, 4, 80, device="cuda", dtype=torch.bfloat16), wide, wide, t, n)
    with pytest.raises(ValueError):
        ops.kv_values(b16)
    with pytest.raises(ValueError, match="power of two"):
        ops.kv_values(kp, 1.5)
    with pytest.raises(ValueError, match="out"):
        ops.kv_values(kp, out=torch.zeros(4, 16, 2, 64, device="cuda"))


def test_launches_are_counted(ops):
    kp, vp = ops.fp4_pages(4, 16, 2, 64), ops.fp4_pages(4, 16, 2, 64)
    k, q = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda", dtype=torch.bfloat16)
    t, n = ints([[0], [1]]), ints([0, 0])
    ops.reset_launch_count()
    ops.kv_append(k, k, kp, vp, t, n)
    ops.prefix_attention(q, kp, vp, t, n)
    ops.kv_values(kp)
    assert ops.launch_count() == 3  # (few keys: attention is one launch)
    ops.prefix_attention(q, kp, vp, t.expand(2, 1).repeat(1, 900), n)
    assert ops.launch_count() == 5


@pytest.mark.parametrize("rows,length", [(1, 90), (3, 2000), (70, 700)])
def test_pages_beyond_four_gigabytes(ops, rows, length):
    """The last of 480,000 pages (4.4 GB of keys and of values): what is appended and read is what a small cache of the same pages gives, bit for bit."""
    many, ps, kv, d, seqs = 480_000, 16, 8, 128, 3
    per = -(-(length + rows) // ps)
    g = torch.Generator(device="cuda").manual_seed(31)
    big = [ops.fp4_pages(many, ps, kv, d) for _ in range(2)]
    small = [torch.randint(256, (seqs * per, kv, 1, 9 * d), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    for s, b in zip(small, big):
        b[many - seqs * per:] = s
    table = torch.arange(seqs * per, dtype=torch.int32, device="cuda").view(seqs, per)
    offsets = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * rows
    lengths = torch.full((seqs,), length, dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(seqs * rows, h, d, generator=g, device="cuda").bfloat16() for h in (32, kv, kv))
    outs = []
    for pages, at in ((big, table + (many - seqs * per)), (small, table)):
        ops.kv_append(k, v, *pages, at, lengths, row_offsets=offsets)
        outs.append(ops.prefix_attention(q, *pages, at, lengths, row_offsets=offsets))
    assert torch.equal(*outs)
    for s, b in zip(small, big):
        assert torch.equal(b[many - seqs * per:], s) and not b[:1000].any()
        assert torch.equal(ops.kv_values(b)[many - seqs * per:], ops.kv_values(s))
