"""verify_drafts without a GPU: its definition and the refusals of the C ABI."""

import ctypes as C

import numpy as np
import pytest

from oracle import verify as V
from velox_voice_b200 import _lib


def test_definition_is_the_targets_distribution():
    """Accepted or redrawn, the first token is distributed as p: summed exactly over all drafts and a grid of random numbers."""
    rng = np.random.default_rng(0)
    x, y = rng.standard_normal((2, 5))
    p, q = (np.exp(t) / np.exp(t).sum() for t in (x, y))
    n, share = 400, np.zeros(5)
    grid = (np.arange(n) + 0.5) / n
    for d in range(5):
        for u in grid:
            if u * q[d] < p[d]:
                share[d] += q[d] / n
            else:
                w = np.maximum(p - q, 0.0)
                share += q[d] / n * w / w.sum()
    assert np.abs(share - p).max() < 2.0 / n
    (a, t, _), = V.verify_ref(np.stack([x, x]), np.array([0, 3]), np.array([[0.0, 0.5], [0.1, 0.999]]), np.stack([y, y]), np.array([0, 2]))
    assert a == 1 and t == V.draw(p, 0.999)


def _desc(**kw):
    d = _lib.VerifyDesc(C.sizeof(_lib.VerifyDesc), _lib.DT_BF16, 6, 100, 2, 4096, 100, 8192, 100, 256, 8, 0, 512, 1024, 1.0, 2048, 2064, 8448, 1 << 20)
    for k, v in kw.items():
        setattr(d, k, v)
    return _lib.load().vx_verify_drafts(C.byref(d), None)


@pytest.mark.parametrize("kw,text", [
    (dict(struct_size=8), b"struct_size"), (dict(reserved=1), b"reserved"), (dict(dtype=9), b"dtype"), (dict(ids_bytes=2), b"ids"), (dict(rows=-1), b"bad shape"),
    (dict(sequences=-1), b"bad shape"), (dict(vocab=0), b"bad shape"), (dict(vocab=2 ** 24 + 1), b"bad shape"), (dict(rows=2 ** 28), b"bad shape"),
    (dict(row_offsets=None), b"row_offsets"), (dict(temperature=-1.0), b"temperature"), (dict(temperature=float("nan")), b"temperature"),
    (dict(temperature=1e-9), b"temperature"), (dict(temperature=float("inf")), b"temperature"), (dict(accepted=None), b"NULL"), (dict(next=None), b"NULL"),
    (dict(logits=None), b"NULL"), (dict(ids=None), b"NULL"), (dict(uniforms=None), b"NULL"), (dict(logits=4097), b"aligned"), (dict(draft_logits=4097), b"aligned"),
    (dict(ids=260), b"aligned"), (dict(uniforms=516), b"aligned"), (dict(ld_logits=99), b"shorter"), (dict(ld_draft=99), b"shorter"), (dict(scratch=None), b"scratch"),
    (dict(scratch_bytes=95), b"scratch"), (dict(scratch=3080), b"scratch")])
def test_argument_errors_come_before_any_launch(kw, text):
    assert _desc(**kw) == -1 and text in _lib.load().vx_last_error()


def test_layout_and_scratch():
    lib = _lib.load()
    assert C.sizeof(_lib.VerifyDesc) == 136 and lib.vx_verify_drafts_scratch(6) == 96 and lib.vx_verify_drafts_scratch(-1) == -1
    assert lib.vx_verify_drafts(None, None) == -1 and _desc(sequences=0, row_offsets=1024) == 0
