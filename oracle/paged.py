"""Paged cache of keys and values and attention over shared prefixes: the definitions, row by row, in fp64.

`kv_append_ref` and `prefix_attention_ref` take numpy arrays laid out as the operators' arguments (caches as fp64 arrays
[pages, page_size, kv_heads, head_dim]) and know nothing of how a kernel splits the work."""

from __future__ import annotations

from typing import Optional

import numpy as np


def row_owner(n_rows: int, n_sequences: int, row_offsets: Optional[np.ndarray]):
    """(sequence, index there) of every row, (-1, 0) where it belongs to none"""
    if row_offsets is None:
        return [(r, 0) for r in range(n_rows)]
    owner = [(-1, 0)] * n_rows
    for s in range(n_sequences):
        for r in range(max(0, row_offsets[s]), min(n_rows, row_offsets[s + 1])):
            owner[r] = (s, r - int(row_offsets[s]))
    return owner


def rotate(x: np.ndarray, angle_row: np.ndarray, interleaved: bool) -> np.ndarray:
    """x [heads, head_dim], angle_row [rot_dim] = cos | sin"""
    rot = angle_row.shape[0]
    c, s = angle_row[:rot // 2], angle_row[rot // 2:]
    y = x.copy()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[:, first] = x[:, first] * c - x[:, second] * s
    y[:, second] = x[:, second] * c + x[:, first] * s
    return y


def _page(table_row: np.ndarray, index: int, pages: int) -> int:
    if index >= table_row.shape[0]:
        return -1
    p = int(table_row[index])
    return p if 0 <= p < pages else -1


def kv_append_ref(q, k, v, k_pages, v_pages, page_table, lengths, rotary=None, interleaved=False, row_offsets=None, starts=None):
    """Returns (q_out, k_pages, v_pages, stored): new arrays, nothing rounded; `stored` bool [pages, page_size] marks the places that
    were written."""
    k_pages, v_pages = k_pages.copy(), v_pages.copy()
    pages, ps = k_pages.shape[:2]
    stored = np.zeros((pages, ps), dtype=bool)
    q_out = None if q is None else np.zeros_like(q)
    for r, (s, i) in enumerate(row_owner(k.shape[0], page_table.shape[0], row_offsets)):
        if s < 0 or lengths[s] < 0:
            continue
        t = int(lengths[s]) + i
        pos = t + (0 if starts is None else int(starts[s]))
        if rotary is not None and not 0 <= pos < rotary.shape[0]:
            continue

        def turned(x):
            return x if rotary is None else rotate(x, rotary[pos], interleaved)

        if q is not None:
            q_out[r] = turned(q[r])
        page = _page(page_table[s], t // ps, pages)
        if page >= 0:
            k_pages[page, t % ps], v_pages[page, t % ps] = turned(k[r]), v[r]
            stored[page, t % ps] = True
    return q_out, k_pages, v_pages, stored


def _run(table_row, n, k_pages, v_pages):
    """keys, values [n', kv_heads, head_dim] and token numbers of the first n tokens, without pages that are not there"""
    pages, ps = k_pages.shape[:2]
    at = [(j, _page(table_row, j // ps, pages)) for j in range(min(int(n), table_row.shape[0] * ps))]
    at = [(j, p) for j, p in at if p >= 0]
    j, p = np.array([a[0] for a in at], dtype=np.int64), np.array([a[1] for a in at], dtype=np.int64)
    return k_pages[p, j % ps], v_pages[p, j % ps], j


def prefix_attention_ref(q, k_pages, v_pages, page_table, lengths, prefix_table=None, prefix_lengths=None, row_offsets=None,
                         group_offsets=None, scale=None):
    """Returns (out, spread) fp64 [rows, heads, head_dim]: the result and sum_j w_j |v_j|, the scale of what rounding the
    probabilities can change."""
    rows, heads, dim = q.shape
    n, kv = page_table.shape[0], k_pages.shape[2]
    per = heads // kv
    scale = dim ** -0.5 if scale is None else scale
    group = np.full(n, -1)
    if prefix_table is not None:
        g = prefix_table.shape[0]
        if group_offsets is None:
            group = np.arange(n) // max(n // g, 1)
        else:
            for e in range(g):
                group[max(0, group_offsets[e]):max(0, group_offsets[e + 1])] = e
        prefix = [_run(prefix_table[e], max(0, int(prefix_lengths[e])), k_pages, v_pages) for e in range(g)]
    out, spread = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    held = {}
    for r, (s, i) in enumerate(row_owner(rows, n, row_offsets)):
        if s < 0 or lengths[s] < 0:
            continue
        if s not in held:
            held = {s: _run(page_table[s], page_table.shape[1] * k_pages.shape[1], k_pages, v_pages)}
        k, v, j = held[s]
        seen = j <= int(lengths[s]) + i
        k, v = k[seen], v[seen]
        if group[s] >= 0:
            k, v = np.concatenate([prefix[group[s]][0], k]), np.concatenate([prefix[group[s]][1], v])
        if k.shape[0] == 0:
            continue
        for h in range(heads):
            x = k[:, h // per] @ q[r, h] * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            out[r, h], spread[r, h] = w @ v[:, h // per], w @ np.abs(v[:, h // per])
    return out, spread
