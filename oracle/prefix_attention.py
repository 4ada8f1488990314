"""CPU restatement of shared-prefix attention in 64 bits, one query token at a time."""

from __future__ import annotations

import numpy as np


def slots_of(table_row, positions, page_size, slots):
    """Slots of ``positions`` in a table row; -1 where there is none inside the planes."""
    index = positions // page_size
    inside = index < len(table_row)
    page = np.where(inside, table_row[np.minimum(index, len(table_row) - 1)] if len(table_row) else -1, -1)
    slot = page.astype(np.int64) * page_size + positions % page_size
    return np.where((page >= 0) & (slot < slots), slot, -1)


def attend(query, k_plane, v_plane, tables, lengths, *, page_size, shared_tokens=0, source_row=0, rows=None,
           query_starts=None, scale=None):
    """Returns (out, lse, weight, reach, seen) for float64 arrays.

    ``weight`` is sum p |v| (what relative errors of p scale with), ``reach`` the largest
    sum_d |scale q_d k_d| over the tokens seen and ``seen`` their number; rows of no request are NaN in ``out``.
    """
    tokens, query_heads, dim = query.shape
    slots, kv_heads, _ = k_plane.shape
    group = query_heads // kv_heads
    batch = len(lengths)
    rows = np.arange(batch) if rows is None else rows
    starts = np.arange(batch + 1) if query_starts is None else query_starts
    scale = dim ** -0.5 if scale is None else scale
    out = np.full(query.shape, np.nan)
    lse = np.full(query.shape[:2], np.nan)
    weight, reach, seen = np.zeros(query.shape), np.zeros(query.shape[:2]), np.zeros(tokens, dtype=np.int64)
    for b in range(batch):
        new = int(starts[b + 1]) - int(starts[b])
        for i in range(new):
            n = int(starts[b]) + i
            visible = max(int(lengths[b]) - new + i + 1, 0)
            position = np.arange(min(visible, tables.shape[1] * page_size))
            row = int(rows[b])
            own = tables[row] if 0 <= row < tables.shape[0] else np.full(tables.shape[1], -1)
            slot = slots_of(own, position, page_size, slots)
            if shared_tokens:
                donor = slots_of(tables[source_row], position, page_size, slots)
                slot = np.where(position < shared_tokens, donor, slot)
            slot = slot[slot >= 0]
            seen[n] = len(slot)
            if not len(slot):
                out[n], lse[n] = 0.0, -np.inf
                continue
            keys, values = k_plane[slot], v_plane[slot]
            for h in range(query_heads):
                k, v = keys[:, h // group], values[:, h // group]
                score = scale * (k @ query[n, h])
                top = score.max()
                p = np.exp(score - top)
                total = p.sum()
                out[n, h] = p @ v / total
                weight[n, h] = p @ np.abs(v) / total
                lse[n, h] = top + np.log(total)
                reach[n, h] = (abs(scale) * (np.abs(k) @ np.abs(query[n, h]))).max()
    return out, lse, weight, reach, seen
