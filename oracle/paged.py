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


# ------------------------------------------------------------------------------------------------ pages in 4 bits

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(1 + b % 8 / 8) * 2.0 ** (b // 8 - 7) if b >= 8 else b * 2.0 ** -9 for b in range(128)])  # (0x7f: 480)


def nearest_even(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the nearest number of an ascending grid, ties to the even index."""
    up = np.clip(np.searchsorted(grid, x), 1, grid.size - 1)
    a, b = x - grid[up - 1], grid[up] - x
    return np.where((a < b) | ((a == b) & ((up - 1) % 2 == 0)), up - 1, up)


def fp4_quantize(x: np.ndarray, g: float = 1.0):
    """Finite fp32 [..., d] -> codes u8 [..., d / 2], scale bytes u8 [..., d / 16]; g: the tensor's scale."""
    assert x.dtype == np.float32
    b = x.astype(np.float64).reshape(*x.shape[:-1], -1, 16) / g
    sixth = (np.abs(b).max(-1) / 6.0).astype(np.float32).astype(np.float64)
    byte = nearest_even(np.minimum(sixth, 448.0), E4M3[:127])
    s = E4M3[byte][..., None]
    q = np.where(s > 0, np.abs(b) / np.where(s > 0, s, 1.0), 0.0)
    code = nearest_even(np.minimum(q, 6.0), E2M1) | ((b < 0) & (s > 0)).astype(np.int64) * 8
    code = code.reshape(x.shape)
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), byte.astype(np.uint8)


def fp4_values(pages: np.ndarray, g: float = 1.0) -> np.ndarray:
    """u8 [pages, kv_heads, units, 9 d] -> fp64 [pages, 16 units, kv_heads, d]"""
    n, kv, units, w = pages.shape
    d = w // 9
    codes = pages[..., :8 * d].reshape(n, kv, units, 16, d // 2)
    codes = np.stack([codes & 15, codes >> 4], -1).reshape(n, kv, units, 16, d)
    scale = E4M3[pages[..., 8 * d:].reshape(n, kv, units, 16, d // 16) & 127]
    x = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0) * np.repeat(scale, 16, -1) * g
    return x.reshape(n, kv, units * 16, d).transpose(0, 2, 1, 3)


def fp4_store(pages: np.ndarray, page: int, token: int, codes: np.ndarray, scales: np.ndarray) -> None:
    """codes [kv_heads, d / 2] and scales [kv_heads, d / 16] of a token into pages, in place"""
    d = pages.shape[3] // 9
    u, t = token // 16, token % 16
    pages[page, :, u, t * (d // 2):(t + 1) * (d // 2)] = codes
    pages[page, :, u, 8 * d + t * (d // 16):8 * d + (t + 1) * (d // 16)] = scales


def rotate_f32(x: np.ndarray, row: np.ndarray, interleaved: bool) -> np.ndarray:
    """`rotate` in fp32, products and sums rounded one by one."""
    rot = row.shape[0]
    c, s = row[:rot // 2], row[rot // 2:]
    y = x.copy()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[:, first] = x[:, first] * c - x[:, second] * s
    y[:, second] = x[:, second] * c + x[:, first] * s
    assert y.dtype == np.float32
    return y


def kv_append_fp4_ref(k, v, k_pages, v_pages, page_table, lengths, rotary=None, interleaved=False, row_offsets=None, starts=None, k_scale=1.0, v_scale=1.0):
    """k, v fp32 [rows, kv_heads, d]; returns new (k_pages, v_pages) bytes."""
    k_pages, v_pages = k_pages.copy(), v_pages.copy()
    pages, ps = k_pages.shape[0], k_pages.shape[2] * 16
    for r, (s, i) in enumerate(row_owner(k.shape[0], page_table.shape[0], row_offsets)):
        if s < 0 or lengths[s] < 0:
            continue
        t = int(lengths[s]) + i
        pos = t + (0 if starts is None else int(starts[s]))
        if rotary is not None and not 0 <= pos < rotary.shape[0]:
            continue
        page = _page(page_table[s], t // ps, pages)
        if page < 0:
            continue
        turned = k[r] if rotary is None else rotate_f32(k[r], rotary[pos], interleaved)
        fp4_store(k_pages, page, t % ps, *fp4_quantize(turned, k_scale))
        fp4_store(v_pages, page, t % ps, *fp4_quantize(v[r], v_scale))
    return k_pages, v_pages
