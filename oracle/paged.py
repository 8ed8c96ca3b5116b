"""NumPy restatement of the operators of a paged Qwen cache (test infrastructure only, see oracle/__init__.py).

The pages, tables and slots are an extension without a counterpart in the reference; norm and rope follow the sequence of
``runtime/qwen/full_attention.py:278-315`` (RMS norm per head, half-split rotary channels) in float64, attention is
``oracle.qwen``'s closed form over the rows that a table names.
"""

from __future__ import annotations

import numpy as np


def page_step(lens, new_lens, tables, free_pages, head, page_size, n_rows):
    """One step, request by request. Returns a dict; ``tables`` and ``free_pages`` in it are the updated copies."""
    lens, tables, stack = list(map(int, lens)), np.array(tables), np.array(free_pages)
    B, width = tables.shape
    cap, top = width * page_size, int(head)
    starts, given, asked_all, taken, placed = [0], [], 0, 0, 0
    for b in range(B):  # given back first, in the order of the requests: request 0's first page ends deepest
        if new_lens[b] < 0:
            given += [int(p) for p in tables[b, :-(-lens[b] // page_size)]]
    top -= len(given)
    stack[top:top + len(given)] = given
    lens_out = []
    slots, positions, visible, requests = (np.full(n_rows, v, dtype=np.int64) for v in (-1, 0, 0, -1))
    for b in range(B):
        asked = max(int(new_lens[b]), 0)
        asked_all += asked
        row0 = min(starts[-1], n_rows)
        rows = min(asked, n_rows - row0)
        starts.append(row0 + rows)
        if new_lens[b] < 0:
            lens_out.append(0)
            continue
        n = lens[b]
        for i in range(rows):
            pos, slot = lens[b] + i, -1
            if n == pos and pos < cap:
                if pos % page_size == 0:
                    if top < len(stack):
                        tables[b, pos // page_size] = stack[top]
                        top, taken = top + 1, taken + 1
                        n += 1
                else:
                    n += 1
                if n > pos:
                    slot = int(tables[b, pos // page_size]) * page_size + pos % page_size
            slots[row0 + i], positions[row0 + i], requests[row0 + i] = slot, pos, b
            visible[row0 + i] = pos + 1 if slot >= 0 else 0
        placed += n - lens[b]
        lens_out.append(n)
    return {"lens": lens_out, "head": [top], "starts": starts, "slots": slots, "positions": positions, "visible": visible,
            "requests": requests, "counts": [asked_all, asked_all - placed, taken, len(given)], "tables": tables,
            "free_pages": stack}


def position_axes(half, sections):
    """The axis of every frequency: 0, 1, 2, 0, 1, 2, ... while the axis has frequencies left, else 0."""
    axes, left = [], list(sections)
    for i in range(half):
        a = i % 3
        if a and i // 3 < left[a]:
            axes.append(a)
        else:
            axes.append(0)
    return axes


def norm_rope(x, weight, positions, inv_freq, eps, sections=None):
    """``x`` [T, H, D]; positions [T] or [3, T]; float64."""
    x = np.asarray(x, dtype=np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)
    half = len(inv_freq)
    pos = np.atleast_2d(np.asarray(positions, dtype=np.float64))
    axes = [0] * half if sections is None else position_axes(half, sections)
    out = y.copy()
    for i in range(half):
        t = pos[axes[i]] * float(inv_freq[i])
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        out[..., i] = y[..., i] * c - y[..., i + half] * s
        out[..., i + half] = y[..., i + half] * c + y[..., i] * s
    return out


def paged_attention(q, keys, values, tables, lens, scale, requests=None):
    """``q`` [R, Hq, D], pages [n, Hkv, page, D] (float64 values of the rows); rows of pages not in the pool are left out."""
    q, n, G, page = np.asarray(q, dtype=np.float64), keys.shape[0], keys.shape[1], keys.shape[2]
    out = np.zeros(q.shape)
    rep = q.shape[1] // G
    for r in range(q.shape[0]):
        b = r if requests is None else int(requests[r])
        if not 0 <= b < len(tables):
            continue
        at = [(int(tables[b][i // page]), i % page) for i in range(min(max(int(lens[r]), 0), len(tables[b]) * page))]
        at = [(p, o) for p, o in at if 0 <= p < n]
        if not at:
            continue
        p, o = (np.array(v) for v in zip(*at))
        for g in range(G):
            k, v = keys[p, g, o].astype(np.float64), values[p, g, o].astype(np.float64)
            s = q[r, g * rep:(g + 1) * rep] @ k.T * scale
            w = np.exp(s - s.max(-1, keepdims=True))
            out[r, g * rep:(g + 1) * rep] = w @ v / w.sum(-1, keepdims=True)
    return out
