"""Edges of the paged cache's arguments that the C entry points decide without a device (descriptors whose pointers are never dereferenced)."""

import ctypes as C

import pytest

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
