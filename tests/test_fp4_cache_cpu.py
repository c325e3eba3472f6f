"""The cache in 4 bits without a GPU: its definition (oracle/paged.py), the refusals of the C ABI and of the operators, what device memory of any content
cannot do."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged as P
from velox_voice_b200 import _lib, ops


def test_nearest_with_ties_to_even_codes():
    x = np.array([0.0, 0.25, 0.2501, 0.75, 0.7499, 1.25, 1.75, 2.5, 2.5001, 3.5, 5.0, 5.001, 6.0])
    assert list(P.E2M1[P.nearest_even(x, P.E2M1)]) == [0, 0, 0.5, 1, 0.5, 1, 2, 2, 3, 4, 4, 6, 6]
    assert P.E4M3[126] == 448 and P.E4M3[8] == 2.0 ** -6 and P.E4M3[1] == 2.0 ** -9


def test_quantization_error_is_bounded():
    """A value is off by half the distance of two codes at most, 1 for the largest: one sixth of the block's largest, more by what the scale is rounded
    (2^-4 of it)."""
    x = np.random.default_rng(0).standard_normal((200, 4, 64)).astype(np.float32)
    codes, scales = P.fp4_quantize(x)
    pages = np.zeros((200, 4, 1, 9 * 64), np.uint8)
    for r in range(200):
        P.fp4_store(pages, r, 3, codes[r], scales[r])
    got = P.fp4_values(pages)[:, 3]
    most = np.abs(x).reshape(200, 4, 4, 16).max(-1).repeat(16, -1)
    assert (np.abs(got - x) <= most / 6 * (1 + 2.0 ** -4) + 1e-9).all()
    assert not P.fp4_values(pages)[:, :3].any()


def _descs():
    """Descriptors whose pointers are never dereferenced."""
    cache = _lib.KvCacheFp4(C.sizeof(_lib.KvCacheFp4), 16, 8, 2, 64, 4096, 8192, 1152, 1152, 1.0, 1.0)
    rows = _lib.KvRows(C.sizeof(_lib.KvRows), 0, 3, 3, 256, None, 512, 4, 4)
    a = _lib.KvAppendDesc(struct_size=C.sizeof(_lib.KvAppendDesc), dtype=_lib.DT_BF16, k=1024, v=2048, k_row=128, k_head=64, v_row=128, v_head=64)
    p = _lib.PrefixAttentionDesc(struct_size=C.sizeof(_lib.PrefixAttentionDesc), q_heads=4, q=1024, q_row=256, q_head=64, out=2048, o_row=256, o_head=64, scale=0.125)
    return cache, rows, a, p


def _refused(rc, text):
    assert rc == -1 and text in _lib.load().vx_last_error(), (rc, _lib.load().vx_last_error())


def test_struct_layout():
    assert C.sizeof(_lib.KvCacheFp4) == 64


@pytest.mark.parametrize("name,pick", [("vx_kv_append_fp4", 2), ("vx_prefix_attention_fp4", 3)])
def test_common_argument_errors_come_before_any_launch(name, pick):
    lib = _lib.load()

    def go(edit=None, null=None):
        d = list(_descs())
        if edit:
            edit(*d)
        args = [C.byref(d[0]), C.byref(d[1]), C.byref(d[pick])]
        if null is not None:
            args[null] = None
        return getattr(lib, name)(*args, None)

    for i, text in enumerate((b"vx_kv_cache_fp4", b"vx_kv_rows", b"struct_size")):
        _refused(go(null=i), text)
    for field, value, text in (("struct_size", 8, b"struct_size"), ("page_size", 0, b"multiple of 16"), ("page_size", 24, b"multiple of 16"),
                               ("pages", 2 ** 31, b"bad shape"), ("pages", -1, b"bad shape"), ("kv_heads", 0, b"bad shape"), ("head_dim", 40, b"head_dim"),
                               ("k", None, b"NULL"), ("v", 8194, b"aligned"), ("k_page", 1160, b"16 bytes apart"), ("v_page", 1136, b"16 bytes apart"),
                               ("k_page", -1152, b"16 bytes apart"), ("k_scale", 3.0, b"powers of two"), ("v_scale", 0.0, b"powers of two"),
                               ("v_scale", float("nan"), b"powers of two"), ("k_scale", float("inf"), b"powers of two"), ("k_scale", -2.0, b"powers of two")):
        _refused(go(lambda c, r, a, p: setattr(c, field, value)), text)
    _refused(go(lambda c, r, a, p: setattr(r, "reserved", 1)), b"reserved")
    _refused(go(lambda c, r, a, p: (setattr(a, "reserved", 1), setattr(p, "reserved", 1))), b"reserved")
    _refused(go(lambda c, r, a, p: setattr(r, "rows", 4)), b"row_offsets")
    _refused(go(lambda c, r, a, p: setattr(r, "lengths", None)), b"lengths")
    _refused(go(lambda c, r, a, p: setattr(r, "ld_table", 3)), b"page_table")


def test_attention_argument_errors():
    lib = _lib.load()

    def go(edit):
        c, r, _, p = _descs()
        edit(c, r, p)
        return lib.vx_prefix_attention_fp4(C.byref(c), C.byref(r), C.byref(p), None)

    _refused(go(lambda c, r, p: (setattr(c, "head_dim", 80), setattr(c, "k_page", 1440), setattr(c, "v_page", 1440))), b"64 or 128")
    _refused(go(lambda c, r, p: setattr(p, "q_heads", 3)), b"multiple")
    for bad in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        _refused(go(lambda c, r, p: setattr(p, "scale", bad)), b"scale")
    _refused(go(lambda c, r, p: (setattr(p, "scale", 1e28), setattr(c, "k_scale", 2.0 ** 32))), b"k_scale")
    _refused(go(lambda c, r, p: setattr(p, "q", None)), b"NULL")
    _refused(go(lambda c, r, p: setattr(p, "o_head", 32)), b"one place")
    _refused(go(lambda c, r, p: (setattr(r, "table_pages", 200), setattr(r, "ld_table", 200))), b"scratch")  # (3,200 keys: parts and a join)


def test_values_argument_errors():
    call = _lib.load().vx_kv_values_fp4
    _refused(call(4096, 2, 1152, 24, 2, 64, 1.0, 256, None), b"multiple of 16")
    _refused(call(4096, 2, 1152, 16, 2, 64, 5.0, 256, None), b"powers of two")
    _refused(call(4096, 2, 1152, 16, 2, 64, 1.0, None, None), b"out")
    _refused(call(4096, 2, 1152, 16, 2, 64, 1.0, 264, None), b"out")
    _refused(call(None, 2, 1152, 16, 2, 64, 1.0, 256, None), b"NULL")
    assert call(None, 0, 0, 16, 2, 64, 1.0, None, None) == 0


def test_pages_are_refused_without_a_gpu():
    for bad in ((-1, 16, 1, 64), (1, 24, 1, 64), (1, 0, 1, 64), (1, 16, 0, 64), (1, 16, 1, 72), (1, 16, 1, 272)):
        with pytest.raises(ValueError):
            ops.fp4_pages(*bad, device="cpu")
    p = ops.fp4_pages(3, 48, 2, 64, device="cpu")
    assert p.shape == (3, 2, 3, 576) and p.dtype == torch.uint8
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv_values(p)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.kv_append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), p, p, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("x", [0.0, 3.0, -1.0, float("nan"), float("inf"), 2.0 ** 33, 2.0 ** -33])
def test_scales_that_are_no_powers_of_two(x):
    with pytest.raises(ValueError, match="power of two"):
        ops._power_of_two(x, "k_scale")
