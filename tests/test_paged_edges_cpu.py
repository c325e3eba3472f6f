"""Edges of the paged cache's arguments that the C entry points decide without a device (descriptors whose pointers are never dereferenced)."""

import ctypes as C
import re
import subprocess

import pytest

from test_device_sources_cpu import source
from test_paged_cpu import _descs, _refused
from velox_voice_b200 import _lib


def attend(edit=None, **kw):
    c, r, _, p = _descs()
    for k, v in kw.items():
        setattr(p, k, v)
    if edit:
        edit(c, r)
    return _lib.load().vx_prefix_attention(C.byref(c), C.byref(r), C.byref(p), None)


# ------------------------------------------------------------------------------------------------ scale


@pytest.mark.parametrize("scale,ok", [(2.3e38, True), (2.4e38, False), (3.0e38, False), (3.3e38, False)])
def test_scales_whose_product_with_log2e_overflows_are_refused(scale, ok):
    """(A scale that is taken comes as far as the check of the scratch.)"""
    _refused(attend(scale=scale), b"scratch" if ok else b"scale")


# ------------------------------------------------------------------------------------------------ rows


def test_rows_of_a_tile_stay_inside_the_run(tmp_path):
    """Offsets that do not ascend can ask for any tile of a run: its first row must not wrap around.  (2^24 owners and more; the function is compiled
    for the host.)"""
    text = source("vx_prefix.cuh")
    body = re.search(r"int first_row\([^{]*\{[^}]*\}", text).group(0)
    src, lib = tmp_path / "first_row.cpp", tmp_path / "first_row.so"
    src.write_text('extern "C" ' + body)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", str(src), "-o", str(lib)], check=True)
    f = C.CDLL(str(lib)).first_row
    assert [f(t, 128, 300) for t in (-1, 0, 1, 2, 3)] == [-1, 0, 128, 256, -1]
    assert [f(t, 8, 8) for t in (0, 1)] == [0, -1] and f(0, 16, 0) == -1 and f(0, 16, -5) == -1
    for tile in (2 ** 24, 2 ** 28, 2 ** 31 - 1, -2 ** 31):
        for tm in (8, 16, 128, 256):
            assert f(tile, tm, 100) == -1 and f(tile, tm, 2 ** 31 - 1) in (-1, tile * tm)
    assert f((2 ** 31 - 2) // 256, 256, 2 ** 31 - 1) == (2 ** 31 - 2) // 256 * 256
    # and it is what both searches take
    assert not re.search(r"rho0 = tile \* ", text) and len(re.findall(r"rho0 = first_row\(", text)) == 2


# ------------------------------------------------------------------------------------------------ results


def test_results_that_share_places_are_refused():
    def append(**kw):
        c, r, a, _ = _descs()
        for k, v in {**dict(q=4096, q_out=8192, q_heads=4, q_row=256, q_head=64, qo_row=256, qo_head=64), **kw}.items():
            setattr(a, k, v)
        return _lib.load().vx_kv_append(C.byref(c), C.byref(r), C.byref(a), None)

    for kw in (dict(qo_row=0), dict(qo_head=0), dict(qo_row=56), dict(qo_head=-8)):
        _refused(append(**kw), b"one place")
    for kw in (dict(o_row=0), dict(o_head=0), dict(o_row=-32), dict(o_head=56)):
        _refused(attend(**kw), b"one place")

    def single(c, r):
        r.rows = r.sequences = 1
        c.kv_heads = 1

    # the stride of a single row or head says nothing
    _refused(attend(single, o_row=0, o_head=0, q_heads=1), b"scratch")


# ------------------------------------------------------------------------------------------------ launches


@pytest.mark.parametrize("rows,sequences,heads,width,prefix,launches", [
    (0, 0, 4, 4, 0, 0),            # nothing
    (3, 0, 4, 4, 0, 1),            # rows of no sequence: zeros
    (3, 3, 4, 0, 0, 1),            # no keys
    (3, 3, 4, 4, 9, 2),            # few rows: both spans in one launch, then the join
    (300, 3, 64, 4, 9, 2),         # prompts: prefix and own tokens in a row, then the rows of no sequence
    (200, 200, 4, 4, 9, 3),        # tile kernel over the prefix, few rows over the own tokens
    (1200, 1200, 4, 4, 900, 3),    # pairs over the prefix
    (60, 3, 8, 16, 9, 2),          # tile kernel over both
    (1600, 80, 8, 16, 900, 3),     # pairs, then slots by themselves
])
def test_launches_of_a_call(rows, sequences, heads, width, prefix, launches):
    c, r, _, p = _descs()
    r.rows, r.sequences, r.ld_table, r.table_pages, r.row_offsets = rows, sequences, max(width, 1), width, 4096
    p.q_heads, p.q_row = heads, 64 * heads
    if prefix:
        p.groups, p.group_offsets, p.prefix_table, p.ld_prefix, p.prefix_pages, p.prefix_lengths = 1, 4096, 4096, prefix, prefix, 8192
    assert _lib.load().vx_prefix_attention_launches(C.byref(c), C.byref(r), C.byref(p)) == launches


def test_launches_of_a_call_that_is_refused():
    c, r, _, p = _descs()
    p.q_heads = 3
    _refused(_lib.load().vx_prefix_attention_launches(C.byref(c), C.byref(r), C.byref(p)), b"multiple")
