"""The error bound by which verify_drafts settles a draft in fp32: its constants, from the source, against the errors of the running sums."""

import re

import pytest

from test_device_sources_cpu import source


@pytest.mark.parametrize("vocab", [1, 5538, 131071, 2 ** 20, 2 ** 22, 2 ** 24])
def test_the_bound_covers_the_errors_of_both_sides(vocab):
    """Each side, u q(d) and p(d) times the other's sum, has an exponential and a sum in it.  An exponential: its exponent, up to 128, is off by 2^-24 of it three times over (the
    difference, log2(e) / T, the product), the instruction by 2^-22: less than 2^-16 of the value.  A thread of a row that is not cut takes at least 16 values at a time; each time its sum is rounded
    (2^-24) and, where the maximum has moved, multiplied by an exponential whose exponent is what it moved by -- those add up to 128 at most, so their errors to 2^-16 once -- and
    which the instruction gives to 2^-22.  The joins of lanes, warps and blocks are eleven more such steps."""
    text = source("vx_verify.cu")
    threads = int(re.search(r"constexpr int VR_THREADS = (\d+);", text).group(1))
    fixed, per_token = (float.fromhex(x) for x in re.search(r"\(0x1p(-\d+)f \+ 0x1p(-\d+)f \* static_cast<float>\(p\.vocab\)\)", text).expand(r"0x1p\1 0x1p\2").split())
    steps = -(-vocab // (16 * threads)) + 11
    side = 2.0 ** -16 + 2.0 ** -16 + 2.0 ** -16 + steps * (2.0 ** -24 + 2.0 ** -22)
    assert 2 * side * (1 + 2.0 ** -8) <= fixed + per_token * vocab
