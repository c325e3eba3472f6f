"""kv_values of more than 2^31 scales: indexes of 64 bits."""

import numpy as np
import pytest
import torch

from test_fp4_cache_gpu import host, ops  # noqa: F401  (ops: the fixture)
from oracle import paged as P

pytestmark = pytest.mark.gpu


def test_values_of_more_than_two_to_the_31_scales(ops):  # noqa: F811
    """2^17 + 3 pages of 16 tokens, 64 heads of 256 (19 GB, 69 GB of values): the first and the last pages and some between hold random bytes, the others zeros."""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    n, kv, d = 2 ** 17 // 16 * 16 + 3, 64, 256
    assert n * 16 * kv * (d // 16) > 2 ** 31
    pages = ops.fp4_pages(n, 16, kv, d)
    at = [0, 1, 65535, 65536, n // 2, n - 2, n - 1]
    x = np.random.default_rng(0).integers(0, 256, (len(at), kv, 1, 9 * d), dtype=np.uint8)
    pages[at] = torch.from_numpy(x).cuda()
    got = ops.kv_values(pages, 0.5)
    assert (host(got[at].double()) == P.fp4_values(x, 0.5)).all()
    for i in range(0, n, 8192):
        assert int(got[i:i + 8192].view(torch.int16).bitwise_and_(0x7fff).ne_(0).any(-1).any(-1).any(-1).sum()) == sum(i <= a < i + 8192 for a in at)
    del pages, got
    torch.cuda.empty_cache()
