"""CPU restatement of the block-table extension and the row append (numpy, request by request)."""

from __future__ import annotations

import numpy as np


def extend(tables, lengths, new_tokens, free_pages, page_size, max_tokens, rows=None):
    """Returns (tables, query_starts, slot_map, positions, lengths, pages_used); ``tables`` is a new array."""
    tables = np.array(tables, dtype=np.int32)
    batch = len(lengths)
    rows = list(range(batch)) if rows is None else [int(r) for r in rows]
    starts, slot_map, positions = [0], [], []
    lengths_out, used, closed = [], 0, False
    for b in range(batch):
        held, new = max(int(lengths[b]), 0), int(new_tokens[b])
        row = rows[b]
        granted = 0
        room = tables.shape[1] * page_size
        if not closed and 0 <= row < tables.shape[0] and new > 0 and held + new <= room:
            had = -(-held // page_size)
            need = -(-(held + new) // page_size) - had
            if used + need > len(free_pages) or len(slot_map) + new > max_tokens:
                closed = True
            else:
                granted = new
                tables[row, had:had + need] = free_pages[used:used + need]
                used += need
                for t in range(held, held + new):
                    page = int(tables[row, t // page_size])
                    slot = page * page_size + t % page_size
                    slot_map.append(slot if page >= 0 and slot < 1 << 31 else -1)
                    positions.append(t)
        starts.append(len(slot_map))
        lengths_out.append(min(held + granted, (1 << 31) - 1))
    pad = [-1] * (max_tokens - len(slot_map))
    as32 = lambda values: np.array(values, dtype=np.int32)  # noqa: E731
    return tables, as32(starts), as32(slot_map + pad), as32(positions + pad), as32(lengths_out), as32([used])


def append(rows, slot_map, plane):
    """``plane`` with ``rows[i]`` at ``slot_map[i]``; slots outside the plane skipped (a new array)."""
    plane = np.array(plane)
    for row, slot in zip(rows, slot_map):
        if 0 <= slot < plane.shape[0]:
            plane[int(slot)] = row
    return plane
