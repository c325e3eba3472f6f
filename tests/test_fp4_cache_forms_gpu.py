"""prefix_attention over a cache in 4 bits, in each form that a call can take: few rows in one launch and in parts, tiles of the
prefix and of own tokens, tiles of up to 64 rows, pairs of tiles with one result and with parts.  In each: scales of the cache, bytes of any kind, queries of all
sizes, scores beyond what fp32 holds to the unit, rows of zeros under tiny scales, probabilities far below the largest.

Tolerances by the number formats, as in test_fp4_cache_gpu.py, but for probabilities far below the row's largest: fp16 holds them to 2^-25 where the largest is
2^7 or more, so they are off by 2^-32 of that, n of them by n 2^-32 of the largest value."""

import math

import numpy as np
import pytest
import torch

from oracle import paged as P
from test_fp4_cache_gpu import ints, host, ops, pages_of, tables  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu

# (heads 4 on 2: two rows per token and key head.)  What decides: rows per owner and key head, how many keys the tables have place for.
FORMS = {
    "whole": dict(rows_of=[1, 2, 1, 3], lengths=[50, 7, 0, 90], prefix=[300]),                       # one launch
    "rows": dict(rows_of=[1, 2, 1, 3], lengths=[1500, 7, 0, 900], prefix=[300]),                     # few rows, in parts
    "rows16": dict(rows_of=[8, 5, 7], lengths=[1500, 7, 900], prefix=[300]),                         # two blocks of eight
    "tiles": dict(rows_of=[5] * 10, lengths=[3 * i for i in range(10)], prefix=[1500]),              # 100 rows over a prefix
    "own": dict(rows_of=[50, 40], lengths=[300, 9]),                                                 # 90 rows over own tokens
    "halves": dict(rows_of=[25, 20, 17], lengths=[400, 30, 0]),                                      # up to 64 rows
    "pairs": dict(rows_of=[100, 70], lengths=[0, 30]),                                               # more than 128, one part
    "parts": dict(rows_of=[100, 70], lengths=[3000, 200], prefix=[100]),                             # in several
    "shared": dict(rows_of=[30] * 10, lengths=[2 * i for i in range(10)], prefix=[900]),             # 600 rows over a prefix
}
EACH = [(f, d) for f in FORMS for d in (64, 128)]


class Call:
    def __init__(self, form, d, *, ps=16, seed=0, heads=4, kv=2, k_scale=1.0, v_scale=1.0, scale=None, pages=None, units=(0x18, 0x31)):
        self.rows_of, self.lengths, prefix = FORMS[form]["rows_of"], FORMS[form]["lengths"], FORMS[form].get("prefix")
        own = [-(-(l + t) // ps) for l, t in zip(self.lengths, self.rows_of)]
        shared = [-(-p // ps) for p in prefix] if prefix else []
        total = sum(own) + sum(shared) + 2
        t, _ = tables(shared + own, total, seed)
        self.pt, self.table = (t[:len(shared)], t[len(shared):]) if shared else (None, t)
        if shared:
            self.pt, self.table = self.pt[:, :max(shared)], self.table[:, :max(own)]
        self.prefix, self.scale, self.k_scale, self.v_scale, self.heads, self.kv, self.d = prefix, scale, k_scale, v_scale, heads, kv, d
        self.kp, self.vp = pages(total, ps, kv, d) if pages else (pages_of(total, ps, kv, d, seed + i, *units) for i in range(2))
        self.off = np.cumsum([0] + self.rows_of)
        self.rows = int(self.off[-1])
        self.q = torch.randn(self.rows, heads, d, generator=torch.Generator().manual_seed(seed))

    def run(self, ops):  # noqa: F811
        from velox_voice_b200 import _lib

        self.q16 = self.q.bfloat16().cuda()
        shared = () if self.pt is None else (ints(self.pt), ints(self.prefix))
        out = ops.prefix_attention(self.q16, torch.from_numpy(self.kp).cuda(), torch.from_numpy(self.vp).cuda(), ints(self.table), ints(self.lengths), *shared,
                                   row_offsets=ints(self.off), scale=self.scale, k_scale=self.k_scale, v_scale=self.v_scale)
        torch.cuda.synchronize()
        assert _lib.device_status() == 0
        return host(out.double())

    def want(self):
        k, v = P.fp4_values(self.kp, self.k_scale), P.fp4_values(self.vp, self.v_scale)
        self.most = np.abs(v).max()
        return P.prefix_attention_ref(host(self.q16.double()), k, v, self.table, np.array(self.lengths), self.pt, None if self.prefix is None else np.array(self.prefix),
                                      self.off, None, self.scale)

    def check(self, ops, small=None):  # noqa: F811
        """`small`: what the rounding of small probabilities can take of a result."""
        out = self.run(ops)
        want, spread = self.want()
        keys = max(l + t for l, t in zip(self.lengths, self.rows_of)) + (max(self.prefix) if self.prefix else 0)
        small = 2.0 ** -32 * keys * self.most if small is None else small
        err = np.abs(out - want)
        bound = 2.0 ** -8 * (np.abs(want) + 2.0 ** -9 * spread) + (2.0 ** -11 + 2.0 ** -13) * spread + small
        assert (err <= bound).all(), f"worst {np.nanmax(err / np.maximum(bound, 1e-300)):.3g} of the tolerance, {(~(err <= bound)).sum()} of {err.size} values, {(~np.isfinite(out)).sum()} not finite"


@pytest.mark.parametrize("form,d", EACH)
@pytest.mark.parametrize("k_scale,v_scale", [(2.0 ** -12, 2.0 ** 9), (2.0 ** 20, 2.0 ** -30)])
def test_scales_of_the_cache(ops, form, d, k_scale, v_scale):  # noqa: F811
    c = Call(form, d, seed=1, k_scale=k_scale, v_scale=v_scale)
    c.q /= k_scale
    c.check(ops)


@pytest.mark.parametrize("form,d", EACH)
def test_any_bytes_are_finite_values(ops, form, d):  # noqa: F811
    c = Call(form, d, seed=2, ps=32, units=(0, 256))
    c.q *= 2.0 ** -9
    c.check(ops)


@pytest.mark.parametrize("form,d", EACH)
def test_queries_of_all_sizes(ops, form, d):  # noqa: F811
    """Rows whose largest values are 2^60 apart, heads of different sizes beside each other, values 2^20 apart in a row, a row of zeros."""
    c = Call(form, d, seed=3)
    c.q *= torch.exp2(torch.linspace(-58, 2, c.rows).round())[:, None, None] * torch.exp2(torch.tensor([0.0, -3.0, -40.0, 0.0]))[:, None]
    c.q[..., ::7] *= 2.0 ** -20
    c.q[c.rows // 2] = 0
    c.check(ops)


@pytest.mark.parametrize("form,d", EACH)
@pytest.mark.parametrize("low", [18, 25, 95])
def test_large_scores(ops, form, d, low):  # noqa: F811
    """One key takes all of the weight; largest scores from 2^18 to 2^110 in units of log2, all sizes between 2^18 and 2^34 among them.  A score in fp32 is off by some
    2^-22 of the largest; rows whose two largest scores are nearer than 2^-18 of that are left out."""
    c = Call(form, d, seed=low)
    c.q *= torch.exp2(low + torch.arange(c.rows) % 11 + 0.15 * torch.arange(4)[:, None] * torch.ones(1, c.rows)).t()[..., None]
    out = c.run(ops)
    assert np.isfinite(out).all()
    k, v, q = P.fp4_values(c.kp), P.fp4_values(c.vp), host(c.q16.double())
    prefix = P._run(c.pt[0], c.prefix[0], k, v)[:2] if c.prefix else (np.zeros((0, 2, d)),) * 2
    compared = 0
    for r, (s, i) in enumerate(P.row_owner(c.rows, len(c.lengths), c.off)):
        ks, vs, _ = P._run(c.table[s], c.lengths[s] + i + 1, k, v)
        ks, vs = np.concatenate([prefix[0], ks]), np.concatenate([prefix[1], vs])
        for h in range(4):
            x = ks[:, h // 2] @ q[r, h] / math.sqrt(d) * math.log2(math.e)
            top = np.sort(x)[-2:]
            if top.size == 1 or top[1] - top[0] > 2.0 ** -18 * np.abs(x).max() + 60:
                compared += 1
                assert np.allclose(out[r, h], vs[x.argmax(), h // 2], rtol=2.0 ** -8, atol=2.0 ** -20), (r, h, np.log2(np.abs(top)), out[r, h], vs[x.argmax(), h // 2])
    assert compared > 3 * c.rows


@pytest.mark.parametrize("form,d", EACH)
@pytest.mark.parametrize("scale,k_scale", [(2.0 ** -60, 1.0), (2.0 ** -30, 2.0 ** -32), (2.0 ** -126, 2.0 ** -32)])
def test_rows_of_zeros_under_a_tiny_scale(ops, form, d, scale, k_scale):  # noqa: F811
    """All scores are 0, more or less: rows are the means of what they see.  (The factor of a row of zeros is below what fp32 holds.)"""
    c = Call(form, d, seed=5, scale=scale, k_scale=k_scale)
    c.q[::3] = 0
    c.check(ops)


def falling(total, ps, kv, d):
    """Units whose first key alone has a score, and a value of 0; the others random values."""
    kp, vp = np.zeros((total, kv, ps // 16, 9 * d), dtype=np.uint8), pages_of(total, ps, kv, d, 6)
    kp[..., 0] = 7                                  # 6 at the first place of the first key
    kp[..., 8 * d:] = 0x38                          # times 1
    vp[..., :d // 2] = 0
    return kp, vp


@pytest.mark.parametrize("form,d", EACH)
@pytest.mark.parametrize("below", [20.0, 24.3, 27.1, 29.0, 31.5])
def test_probabilities_far_below_the_largest(ops, form, d, below):  # noqa: F811
    """Every unit has a key with the row's largest score and a value of 0; the others, which alone have values, are `below` powers of two less likely.  A row that
    sees n keys sees n / 16 of the former or more, so the largest share is 16 / n, and what is lost 16 2^-32 of the largest value at most."""
    c = Call(form, d, seed=7, pages=falling, scale=below * math.log(2) / 6)
    c.q[:] = 0
    c.q[..., 0] = 1
    c.check(ops, small=16 * 2.0 ** -32 * np.abs(P.fp4_values(c.vp)).max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [90_000, 1_000_000])
@pytest.mark.parametrize("below", [20.1, 25.1, 28.1, 31.0])
@pytest.mark.parametrize("rows", [1, 50, 100, 200])
def test_one_key_in_front_of_a_long_tail(ops, d, n, below, rows):  # noqa: F811
    """The first key has a value of 0, n others, each `below` powers of two less likely, a value of 1.  (The rows are one sequence's, whose own tokens are of the tail.)  fp32
    sums of up to n equal numbers, some 2^14 of them one after another: 2^-10 of the result."""
    ps = 16
    kp, vp = np.zeros((2, 1, 1, 9 * d), dtype=np.uint8), np.full((2, 1, 1, 9 * d), 0x22, dtype=np.uint8)
    kp[..., 8 * d:] = vp[..., 8 * d:] = 0x38
    kp[0, ..., 0] = 7
    vp[0, ..., :d // 2] = 0
    q = torch.zeros(rows, 1, d, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1
    table = torch.ones(1, n // ps, dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    out = ops.prefix_attention(q, torch.from_numpy(kp).cuda(), torch.from_numpy(vp).cuda(), ints([[1] * -(-rows // ps)]), ints([0]), table, ints([n]), row_offsets=ints([0, rows]),
                               scale=below * math.log(2) / 6)
    tail = (n - 1 + 1 + np.arange(rows)) * 2.0 ** -below
    want = (tail / (1 + tail))[:, None, None]
    assert (np.abs(host(out.double()) - want) <= want * (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -13) + 2.0 ** -32 * n).all(), (host(out.double()).min() / want.min(), host(out.double()).max() / want.max())


def test_a_scale_below_the_normal_numbers(ops):  # noqa: F811
    """scale 2^-149 with k_scale 2^32: their product with log2(e) is formed before it is rounded."""
    d, ps = 64, 16
    c = Call("whole", d, seed=8, scale=2.0 ** -149, k_scale=2.0 ** 32)
    c.q *= 2.0 ** 112
    c.check(ops)


@pytest.mark.parametrize("form,d", EACH)
@pytest.mark.parametrize("low", [-100, -118, -124])
def test_queries_below_2_to_the_minus_100(ops, form, d, low):  # noqa: F811
    """Down to the smallest numbers of bf16, under a scale that makes scores of them (2^84 log2(e) times 256 times k_scale is the largest that is taken)."""
    c = Call(form, d, seed=9, scale=2.0 ** min(-low - 34, 84), k_scale=2.0 ** 32, units=(0x18, 0x31) if low > -120 else (0x40, 0x51))
    c.q *= 2.0 ** low
    c.q[1::5] *= 2.0 ** -6
    c.check(ops)
