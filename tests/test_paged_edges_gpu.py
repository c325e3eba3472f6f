"""kv_append and prefix_attention at the edges of their arguments: tables without rows, offsets in front of the call's rows, scores that are
large numbers, tables whose rows are one row.

Tolerances are those of test_paged_gpu.py; where nothing is rounded the results are compared bit by bit."""

import pytest
import torch

from test_paged_gpu import ints, make_cache, ops  # noqa: F401

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
