"""The paged cache without a device: the oracle against an independent formula, argument errors of the C ABI before any launch, and
the operators' checks of tensors that are not on a GPU."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged as P
from velox_voice_b200 import _lib, ops


def test_rotary_table():
    t = ops.rotary_table(50, 32, 100.0, device="cpu")
    assert t.shape == (50, 32) and t.dtype == torch.float32
    p, i = 37, 5
    assert abs(t[p, i].item() - np.cos(p * 100.0 ** (-2 * i / 32))) < 2 ** -24 and abs(t[p, 16 + i].item() - np.sin(p * 100.0 ** (-2 * i / 32))) < 2 ** -24
    with pytest.raises(ValueError):
        ops.rotary_table(5, 24, device="cpu")


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation_keeps_relative_positions(interleaved):
    """The product of a rotated query and a rotated key depends on the difference of their positions; the length stays."""
    rng = np.random.default_rng(0)
    t = ops.rotary_table(60, 32, device="cpu").double().numpy()
    q, k = rng.standard_normal((2, 1, 48))
    dots = [float((P.rotate(q, t[a], interleaved) * P.rotate(k, t[a + 7], interleaved)).sum()) for a in (0, 11, 40)]
    assert np.allclose(dots, dots[0], atol=1e-5) and not np.isclose(dots[0], (q * k).sum())
    assert np.isclose((P.rotate(q, t[9], interleaved) ** 2).sum(), (q ** 2).sum(), atol=1e-5)
    assert (P.rotate(q, t[9], interleaved)[:, 32:] == q[:, 32:]).all()


def test_oracle_attention_equals_a_masked_softmax():
    rng = np.random.default_rng(1)
    ps, kv, per, d, n, prefix = 4, 2, 3, 8, 3, 11
    table = np.array([[0, 1, 2, 3], [4, 5, -1, 6], [7, 8, 9, 10]])
    ptable = np.array([[11, 12, 13]])
    k, v = rng.standard_normal((2, 14, ps, kv, d))
    lengths, off = np.array([3, 9, -1]), np.array([1, 6, 7, 9])
    q = rng.standard_normal((10, kv * per, d))
    out, _ = P.prefix_attention_ref(q, k, v, table, lengths, ptable, [prefix], off, [0, n])
    assert not out[[0, 7, 8, 9]].any()
    for r in range(1, 7):
        s = 0 if r < 6 else 1
        own = torch.from_numpy(k[table[s]].reshape(-1, kv, d)), torch.from_numpy(v[table[s]].reshape(-1, kv, d))
        pre = torch.from_numpy(k[ptable[0]].reshape(-1, kv, d)[:prefix]), torch.from_numpy(v[ptable[0]].reshape(-1, kv, d)[:prefix])
        j = np.arange(16)
        seen = torch.from_numpy(np.concatenate([np.ones(prefix, bool), (j <= lengths[s] + r - off[s]) & (table[s][j // ps] >= 0)]))
        keys, vals = torch.cat([pre[0], own[0]]), torch.cat([pre[1], own[1]])
        x = torch.einsum("hd,jhd->hj", torch.from_numpy(q[r]), keys.repeat_interleave(per, 1)) / d ** 0.5
        w = torch.softmax(x.masked_fill(~seen, float("-inf")), -1)
        want = torch.einsum("hj,jhd->hd", w, vals.repeat_interleave(per, 1))
        assert np.allclose(out[r], want.numpy(), atol=1e-12)


def test_oracle_append_and_attend_by_steps_equal_one_chunk():
    rng = np.random.default_rng(2)
    ps, kv, d, t = 4, 1, 8, 10
    table, cache = np.array([[2, 0, 1]]), np.zeros((2, 3, ps, kv, d))
    q, k, v = rng.standard_normal((3, t, kv, d))
    _, kc, vc, stored = P.kv_append_ref(q, k, v, *cache, table, np.array([0]), row_offsets=np.array([0, t]))
    assert stored.sum() == t
    whole, _ = P.prefix_attention_ref(q, kc, vc, table, np.array([0]), row_offsets=np.array([0, t]))
    kc, vc = cache
    for i in range(t):
        _, kc, vc, _ = P.kv_append_ref(None, k[i:i + 1], v[i:i + 1], kc, vc, table, np.array([i]))
        one, _ = P.prefix_attention_ref(q[i:i + 1], kc, vc, table, np.array([i]))
        assert np.allclose(one[0], whole[i], atol=1e-12)


# ------------------------------------------------------------------------------------------------ C ABI


def _descs():
    """Descriptors whose pointers are never dereferenced."""
    cache = _lib.KvCache(C.sizeof(_lib.KvCache), 16, 8, 2, 64, 4096, 8192, 2048, 128, 64, 2048, 128, 64)
    rows = _lib.KvRows(C.sizeof(_lib.KvRows), 0, 3, 3, 256, None, 512, 4, 4)
    a = _lib.KvAppendDesc(struct_size=C.sizeof(_lib.KvAppendDesc), dtype=_lib.DT_BF16, k=1024, v=2048, k_row=128, k_head=64, v_row=128, v_head=64)
    p = _lib.PrefixAttentionDesc(struct_size=C.sizeof(_lib.PrefixAttentionDesc), q_heads=4, q=1024, q_row=256, q_head=64, out=2048, o_row=256, o_head=64, scale=0.125)
    return cache, rows, a, p


def _refused(rc, text):
    assert rc == -1 and text in _lib.load().vx_last_error(), (rc, _lib.load().vx_last_error())


def test_struct_layouts():
    assert [C.sizeof(t) for t in (_lib.KvCache, _lib.KvRows, _lib.KvAppendDesc, _lib.PrefixAttentionDesc)] == [88, 64, 152, 128]


def test_common_argument_errors_come_before_any_launch():
    lib = _lib.load()
    for call, pick in ((lib.vx_kv_append, 2), (lib.vx_prefix_attention, 3)):
        def go(edit=None, null=None):
            d = list(_descs())
            if edit:
                edit(*d)
            args = [C.byref(d[0]), C.byref(d[1]), C.byref(d[pick])]
            if null is not None:
                args[null] = None
            return call(*args, None)

        for i, text in enumerate((b"vx_kv_cache", b"vx_kv_rows", b"struct_size")):
            _refused(go(null=i), text)
        _refused(go(lambda c, r, a, p: setattr(c, "struct_size", 8)), b"vx_kv_cache: struct_size")
        _refused(go(lambda c, r, a, p: setattr(r, "struct_size", 8)), b"vx_kv_rows: struct_size")
        _refused(go(lambda c, r, a, p: (setattr(a, "struct_size", 8), setattr(p, "struct_size", 8))), b"struct_size")
        _refused(go(lambda c, r, a, p: (setattr(a, "reserved", 1), setattr(p, "reserved", 1))), b"reserved")
        _refused(go(lambda c, r, a, p: setattr(r, "reserved", 1)), b"reserved")
        _refused(go(lambda c, r, a, p: setattr(c, "page_size", 0)), b"bad shape")
        _refused(go(lambda c, r, a, p: setattr(c, "pages", 2 ** 31)), b"bad shape")
        _refused(go(lambda c, r, a, p: setattr(c, "kv_heads", 0)), b"bad shape")
        _refused(go(lambda c, r, a, p: setattr(c, "k", None)), b"NULL")
        _refused(go(lambda c, r, a, p: setattr(c, "v", 8194)), b"aligned")
        _refused(go(lambda c, r, a, p: setattr(c, "v_token", 12)), b"multiples of 8")
        _refused(go(lambda c, r, a, p: setattr(c, "k_head", -64)), b"multiples of 8")
        _refused(go(lambda c, r, a, p: setattr(r, "rows", 4)), b"row_offsets")
        _refused(go(lambda c, r, a, p: setattr(r, "rows", -1)), b"bad shape")
        _refused(go(lambda c, r, a, p: setattr(r, "lengths", None)), b"lengths")
        _refused(go(lambda c, r, a, p: setattr(r, "page_table", None)), b"page_table")
        _refused(go(lambda c, r, a, p: setattr(r, "ld_table", 3)), b"page_table")
        _refused(go(lambda c, r, a, p: (setattr(r, "ld_table", 2 ** 28), setattr(r, "table_pages", 2 ** 28))), b"2^31")


def test_append_argument_errors():
    lib = _lib.load()

    def go(edit=None, **kw):
        c, r, a, _ = _descs()
        for k, v in kw.items():
            setattr(a, k, v)
        if edit:
            edit(c, r)
        return lib.vx_kv_append(C.byref(c), C.byref(r), C.byref(a), None)

    _refused(go(lambda c, r: setattr(c, "head_dim", 40)), b"head_dim")
    _refused(go(lambda c, r: setattr(c, "head_dim", 272)), b"head_dim")
    _refused(go(lambda c, r: setattr(c, "k_page", 0)), b"one place")
    _refused(go(lambda c, r: setattr(c, "v_token", 0)), b"one place")
    _refused(go(lambda c, r: setattr(c, "k_head", 0)), b"one place")
    _refused(go(dtype=_lib.DT_FP4), b"dtype")
    _refused(go(k=None), b"NULL")
    _refused(go(k=1026), b"aligned")
    _refused(go(v_row=130), b"aligned")
    _refused(go(q=4096), b"together")
    _refused(go(q_out=4096), b"together")
    _refused(go(q=4096, q_out=8192, q_heads=0), b"together")
    _refused(go(q=4096, q_out=8192, q_heads=4, q_row=256, q_head=64, qo_row=256, qo_head=60), b"aligned")
    _refused(go(q=4096, q_out=4096, q_heads=4, q_row=256, q_head=64, qo_row=512, qo_head=64), b"q_out may be q")
    _refused(go(q=4096, q_out=4096, q_heads=4, q_row=256, q_head=64, qo_row=256, qo_head=64, dtype=_lib.DT_F32), b"q_out may be q")
    for bad in (0, 24, 80):
        _refused(go(rotary=4096, positions=9, ld_rotary=128, rot_dim=bad), b"rot_dim")
    _refused(go(rotary=4096, positions=9, ld_rotary=32, rot_dim=64), b"rotary")
    _refused(go(rotary=4100, positions=9, ld_rotary=64, rot_dim=64), b"rotary")

    def empty(c, r):
        r.rows = r.sequences = 0

    assert go(empty) == 0 and go(empty, k=None, v=None) == 0


def test_attention_argument_errors():
    lib = _lib.load()

    def go(edit=None, scratch=False, **kw):
        c, r, _, p = _descs()
        for k, v in kw.items():
            setattr(p, k, v)
        if edit:
            edit(c, r)
        if scratch:
            return lib.vx_prefix_attention_scratch(C.byref(c), C.byref(r), C.byref(p))
        return lib.vx_prefix_attention(C.byref(c), C.byref(r), C.byref(p), None)

    _refused(go(lambda c, r: setattr(c, "head_dim", 96)), b"head_dim")
    _refused(go(q_heads=3), b"multiple")
    _refused(go(q_heads=0), b"multiple")
    _refused(go(q=None), b"NULL")
    _refused(go(out=None), b"NULL")
    _refused(go(q=1032), b"aligned")
    _refused(go(o_head=68), b"aligned")
    _refused(go(groups=-1), b"groups")
    prefix = dict(groups=1, prefix_table=4096, ld_prefix=9, prefix_pages=9, prefix_lengths=8192)
    _refused(go(**{**prefix, "groups": 2}), b"group_offsets")
    _refused(go(**{**prefix, "prefix_lengths": None}), b"prefix_lengths")
    _refused(go(**{**prefix, "prefix_table": None}), b"prefix_lengths")
    _refused(go(**{**prefix, "ld_prefix": 8}), b"prefix_lengths")
    _refused(go(**{**prefix, "prefix_pages": 2 ** 28, "ld_prefix": 2 ** 28}), b"2^31")

    def many(c, r):
        r.rows, r.row_offsets = 2 ** 29, 4096

    _refused(go(many), b"2^31")

    def wide(c, r):
        r.table_pages = r.ld_table = 2 ** 26

    def wider(c, r):
        r.table_pages = r.ld_table = 2 ** 60

    _refused(go(wide, **{**prefix, "prefix_pages": 2 ** 27 - 2 ** 26, "ld_prefix": 2 ** 27}), b"together")
    _refused(go(wider), b"2^31")
    _refused(go(**{**prefix, "prefix_pages": 2 ** 60, "ld_prefix": 2 ** 60}), b"2^31")
    _refused(go(**{**prefix, "groups": 2 ** 31 - 1, "group_offsets": 4096}), b"2^31")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        _refused(go(scale=bad), b"scale")
    need = go(scratch=True)
    assert need > 0 and need % 32 == 0

    def at(address, size):  # of the scratch
        c, r, _, p = _descs()
        p.scratch, p.scratch_bytes = address, size
        return lib.vx_prefix_attention(C.byref(c), C.byref(r), C.byref(p), None)

    _refused(at(None, need), b"scratch")
    _refused(at(4096 + 16, need), b"scratch")
    _refused(at(4096, need - 1), b"scratch")
    assert go(scratch=True, q_heads=3) == -1

    def empty(c, r):
        r.rows = r.sequences = 0

    assert go(empty) == 0 and go(empty, q=None, out=None) == 0 and go(empty, scratch=True) == 0


def test_operators_have_no_cpu_path():
    k = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.kv_append(k, k, pages, pages, t, n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.prefix_attention(k, pages, pages, t, n)
