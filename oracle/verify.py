"""Verification of drafted tokens, row by row in fp64."""

from __future__ import annotations

from typing import Optional

import numpy as np


def _softmax(x: np.ndarray, t: float) -> Optional[np.ndarray]:
    """None: nothing finite, NaN or +infinity"""
    if np.isnan(x).any() or np.isposinf(x).any() or not np.isfinite(x).any():
        return None
    w = np.exp((x - x.max()) / t)
    return w / w.sum()


def draw(w: np.ndarray, u: float) -> int:
    c = np.cumsum(w)
    return int(np.argmax(c > u * c[-1]))


def border(w: np.ndarray, u: float) -> float:
    """How far u is from the nearest border between two tokens, as a share of all."""
    c = np.cumsum(w) / w.sum()
    return float(np.abs(c - u).min())


def verify_ref(logits, ids, uniforms, draft_logits=None, row_offsets=None, temperature=1.0):
    """fp64 [rows, vocab], ints [rows], fp64 [rows, 2] -> [(accepted, next, margin)] per sequence; margin: how near any of its comparisons came to its border
    (relative), infinite for temperature 0"""
    rows, vocab = logits.shape
    off = np.arange(rows + 1) if row_offsets is None else np.clip(row_offsets, 0, rows)
    out = []
    for r0, r1 in zip(off[:-1], off[1:]):
        n, margin = r1 - r0 - 1, np.inf
        if n < 0:
            out.append((0, -1, margin))
            continue
        i, token = 0, -1
        while True:
            r = r0 + i
            d = int(ids[r + 1]) if i < n else -1
            if temperature == 0.0:
                x = logits[r]
                best = int(np.argmax(x)) if not np.isnan(x).any() and np.isfinite(x.max()) else -1
                if i < n and best >= 0 and best == d:
                    i += 1
                    continue
                token = best
                break
            p = _softmax(logits[r], temperature)
            q = None
            if i < n:
                if draft_logits is not None:
                    q = _softmax(draft_logits[r], temperature)
                else:
                    q = np.zeros(vocab)
                    if 0 <= d < vocab:
                        q[d] = 1.0
            if p is None or (i < n and q is None):
                break
            if i < n and 0 <= d < vocab:
                left, right = uniforms[r, 0] * q[d], p[d]
                margin = min(margin, abs(left - right) / max(left, right, 1e-300))
                if left < right:
                    i += 1
                    continue
            w = p if i == n else np.maximum(p - q, 0.0)
            if not w.sum() > 0:
                w = p
            margin = min(margin, border(w, uniforms[r, 1]))
            token = draw(w, uniforms[r, 1])
            break
        out.append((i, token, margin))
    return out
