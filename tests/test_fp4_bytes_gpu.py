"""kv_append into a cache in 4 bits where the largest of 16 values is beyond what a scale can bring to 6: bytes as defined (oracle/paged.py)."""

import numpy as np
import pytest
import torch

from test_fp4_cache_gpu import check_append, host, ints, ops  # noqa: F401  (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("largest", [2688.0, 1e29, 1e30, 3e30, -3.0e38, 3.4028234663852886e38])
@pytest.mark.parametrize("g", [1.0, 2.0 ** -9, 2.0 ** 9])
def test_values_beside_a_very_large_one(ops, largest, g):  # noqa: F811
    """The scale is 448 g; the neighbours of the borders between codes, 448 g (0.25, 0.75, ...), go to the code of the exact quotient."""
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32) * np.float32(448 * g)
    near = np.stack([border, np.nextafter(border, np.float32(0)), np.nextafter(border, np.float32(np.inf))], 1)
    assert {783.99994, 1567.9999} <= {round(float(x) / g, 5) for x in near.flatten()} | {round(float(x) / g, 4) for x in near.flatten()}

    def edit(x):
        rows = torch.zeros(42, 64)
        for r in range(42):
            b = torch.from_numpy(np.roll(near.flatten(), r)[:15].copy()) * (-1) ** (r // 21)
            for i in range(4):
                rows[r, 16 * i:16 * i + 15], rows[r, 16 * i + 15] = b.roll(i), largest
        x[:, -64:] = x[:, -192:-128] = rows.cuda()

    check_append(ops, rows_of=[42], lengths=[0], kv=2, edit=edit, dtype=torch.float32, rot=0, k_scale=g, v_scale=g)


def test_values_beside_an_infinity(ops):  # noqa: F811
    """Infinities are stored as the largest values of their signs, their neighbours by the exact quotient by 448."""
    x = torch.zeros(2, 1, 64, device="cuda")
    x[:, 0, :6] = torch.tensor([783.99994, 784.0, 1567.9999, 1568.0, -112.0, 112.00001])
    x[0, 0, 9], x[1, 0, 9], x[1, 0, 10] = float("inf"), float("-inf"), 1e31
    kp, vp = ops.fp4_pages(1, 16, 1, 64), ops.fp4_pages(1, 16, 1, 64)
    ops.kv_append(x, x.clone(), kp, vp, ints([[0]]), ints([0]), row_offsets=ints([0, 2]))
    want = [672.0, 896.0, 1344.0, 1792.0, 0.0, 224.0]
    for p in (kp, vp):
        got = host(ops.kv_values(p).double())[0, :2, 0]
        assert (got[:, :6] == want).all() and got[0, 9] == 2688 and got[1, 9] == -2688 and got[1, 10] == 2688 and not got[:, 11:].any()


def test_not_a_number_beside_values(ops):  # noqa: F811
    """What stands for NaN is any finite value; the scale is that of the other values."""
    x = torch.zeros(1, 1, 64, device="cuda")
    x[0, 0, :4] = torch.tensor([6.0, float("nan"), 3.0, -1.5])
    kp, vp = ops.fp4_pages(1, 16, 1, 64), ops.fp4_pages(1, 16, 1, 64)
    ops.kv_append(x, x.clone(), kp, vp, ints([[0]]), ints([0]))
    got = host(ops.kv_values(vp).double())[0, 0, 0]
    assert np.isfinite(got).all() and got[0] == 6 and got[2] == 3 and got[3] == -1.5 and not got[4:].any()
