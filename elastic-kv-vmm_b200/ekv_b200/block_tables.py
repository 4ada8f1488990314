"""Block tables, slot maps and the row append of a serving step.

``extend_block_tables`` gives the new tokens of a step their places: from the requests'
lengths alone it takes the pages they need from a list of free ones, enters them in the
block table and writes, for every new token, its slot and its position -- in one launch,
without reading anything back, so it also runs inside a captured graph.  ``append_rows``
then writes the tokens' K and V rows to those slots of the pool planes.

A block table is an int32 ``[rows, width]`` tensor: entry ``[r, i]`` is the page that
holds positions ``i * page_size .. (i + 1) * page_size - 1`` of table row ``r``, and the
slot of a position is ``page * page_size + position % page_size``.  At page size 1 it is a
request table of slots.  Nothing here has a counterpart in the reference, whose engine's
allocator hands out slots on the host.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import MAX_PLANES, call, index_esize, last_error, require_cuda, stream_handle, torch_binding, u64_array

_INT32_MAX = (1 << 31) - 1


class TableExtension(NamedTuple):
    """What ``extend_block_tables`` writes (int32, contiguous).

    ``query_starts`` [B + 1]: request b's new tokens are ``query_starts[b]`` up to
    ``query_starts[b + 1]``; ``slot_map`` and ``positions`` [max_tokens]: slot and position
    of each, -1 behind the last; ``lengths`` [B]: the lengths with the granted tokens;
    ``pages_used`` [1]: pages taken from the front of ``free_pages``.
    """

    query_starts: torch.Tensor
    slot_map: torch.Tensor
    positions: torch.Tensor
    lengths: torch.Tensor
    pages_used: torch.Tensor


def _vector(tensor: torch.Tensor, name: str, count: int | None) -> int:
    """Element size of a contiguous one-dimensional index tensor (``count`` entries if given)."""
    if tensor.dim() != 1 or (tensor.numel() > 1 and tensor.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous one-dimensional tensor")
    if count is not None and tensor.shape[0] != count:
        raise ValueError(f"{name} must have {count} entries")
    return index_esize(tensor, name)


def _end(tensor: torch.Tensor) -> int:
    last = sum((n - 1) * s for n, s in zip(tensor.shape, tensor.stride()))
    return tensor.data_ptr() + (last + 1) * tensor.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    return bool(a.numel() and b.numel()) and a.data_ptr() < _end(b) and b.data_ptr() < _end(a)


def extend_block_tables(block_tables: torch.Tensor, lengths: torch.Tensor, new_tokens: torch.Tensor,
                        free_pages: torch.Tensor, *, page_size: int, max_tokens: int,
                        rows: torch.Tensor | None = None, out: TableExtension | None = None) -> TableExtension:
    """Pages and slots for ``new_tokens[b]`` more tokens of each request of a batch.

    ``lengths`` [B] are the tokens that the requests hold, ``rows`` [B] their rows of
    ``block_tables`` (default: request b is row b; a negative or too large row gets
    nothing, as does ``new_tokens[b] <= 0``).  Pages are taken from ``free_pages`` [F] in
    order.  Requests are granted in batch order until one needs more pages than are left
    or more tokens than ``max_tokens`` holds; it and all after it get nothing, which shows
    in the returned lengths.  A request whose tokens its table row cannot hold is passed over.
    A negative page, in the table or in ``free_pages``, gives its tokens slot -1.

    Tokens that fill up a request's last page go to the page that its row names there.  A request that
    begins with shared tokens which end inside a page must therefore have a page of its own in that entry:
    with none its tokens get slot -1, and with the donor's all requests would write into that one.

    ``block_tables`` is written in place (only the entries of taken pages); nothing else
    among the inputs changes, so the step can be repeated.  Active requests must have
    distinct rows, and no other input may lie in the entries that are written.  ``out`` takes the tensors of an earlier result again; they must not
    overlap the inputs or one another (copy ``out.lengths`` to the next step's lengths instead).
    """
    fast = torch_binding() if out is None and type(page_size) is int and type(max_tokens) is int else None
    if fast is not None:
        try:
            rc, *results = fast.extend_block_tables(block_tables, lengths, new_tokens, free_pages, page_size, max_tokens, rows)
        except TypeError:  # not tensors: the checked path below reports it
            rc = fast.NOT_HANDLED
        if rc == 0:
            return TableExtension(*results)
        if rc == fast.KERNEL_ERROR:
            raise last_error("ekv_extend_block_tables")
    if type(page_size) is not int or not 1 <= page_size <= _INT32_MAX:
        raise ValueError("page_size outside the supported range")
    if type(max_tokens) is not int or not 0 <= max_tokens <= _INT32_MAX:
        raise ValueError("max_tokens outside the supported range")
    device = require_cuda(dict(block_tables=block_tables, lengths=lengths, new_tokens=new_tokens,
                               free_pages=free_pages, rows=rows))
    if block_tables.dtype != torch.int32 or free_pages.dtype != torch.int32:
        raise TypeError("block_tables and free_pages must be int32 tensors")
    if block_tables.dim() != 2 or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [rows, width] with contiguous rows")
    if block_tables.shape[0] > 1 and block_tables.stride(0) < block_tables.shape[1]:
        raise ValueError("block_tables rows overlap")
    if block_tables.shape[1] * page_size > _INT32_MAX:
        raise ValueError("a table row covers more than 2^31 - 1 positions")
    batch = lengths.shape[0] if lengths.dim() == 1 else -1
    len_es = _vector(lengths, "lengths", None)
    new_es = _vector(new_tokens, "new_tokens", batch)
    rows_es = 8 if rows is None else _vector(rows, "rows", batch)
    _vector(free_pages, "free_pages", None)
    if out is None:
        # One allocation for the five outputs.
        flat = torch.empty(2 * batch + 2 * max_tokens + 2, dtype=torch.int32, device=device)
        out = TableExtension(*flat.split([batch + 1, max_tokens, max_tokens, batch, 1]))
    else:
        inputs = [t for t in (block_tables, lengths, new_tokens, free_pages, rows) if t is not None]
        for tensor, name, count in zip(out, TableExtension._fields, (batch + 1, max_tokens, max_tokens, batch, 1)):
            require_cuda({name: tensor}, device)
            if tensor.dtype != torch.int32:
                raise TypeError(f"{name} must be an int32 tensor")
            _vector(tensor, name, count)
            if any(_overlap(tensor, t) for t in inputs):
                raise ValueError(f"{name} overlaps an input")
        spans = sorted((tensor.data_ptr(), _end(tensor)) for tensor in out if tensor.numel())
        if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("the tensors of out overlap")
    call(
        "ekv_extend_block_tables",
        block_tables.data_ptr(), block_tables.shape[0], block_tables.shape[1], block_tables.stride(0),
        None if rows is None else rows.data_ptr(), rows_es,
        lengths.data_ptr(), len_es, new_tokens.data_ptr(), new_es, batch,
        free_pages.data_ptr(), free_pages.shape[0], page_size, max_tokens,
        out.query_starts.data_ptr(), out.slot_map.data_ptr(), out.positions.data_ptr(),
        out.lengths.data_ptr(), out.pages_used.data_ptr(), device.index, stream_handle(device),
    )
    return out


def _row_stride(tensor: torch.Tensor, name: str) -> int:
    """Elements between the rows of ``[count, ...]``; each row must be contiguous."""
    expected = 1
    for size, stride in zip(reversed(tensor.shape[1:]), reversed(tensor.stride()[1:])):
        if size != 1 and stride != expected:
            raise ValueError(f"{name} must have contiguous rows")
        expected *= size
    return tensor.stride(0) if tensor.shape[0] > 1 else expected


def append_rows(rows, slot_map: torch.Tensor, planes) -> None:
    """Write ``rows[p][i]`` to slot ``slot_map[i]`` of ``planes[p]``, for every plane p.

    ``rows[p]`` is ``[tokens, ...]`` and ``planes[p]`` ``[slots, ...]`` with the same row
    shape and dtype (e.g. the new tokens' K and V, and a layer's K and V planes).  Rows are
    contiguous within; all ``rows`` share one stride between tokens and all ``planes`` one
    between slots, so the views of a fused projection need no copy.  Tokens whose slot is
    negative or not below ``slots`` are skipped; slots must be distinct, planes too, and
    ``rows`` must not lie in them.  The payload is copied bit for bit.
    """
    rows, planes = list(rows), list(planes)
    fast = torch_binding()
    if fast is not None:
        try:
            rc = fast.append_rows(rows, slot_map, planes)
        except TypeError:  # not tensors: the checked path below reports it
            rc = fast.NOT_HANDLED
        if rc == 0:
            return
        if rc == fast.KERNEL_ERROR:
            raise last_error("ekv_append_rows")
    if len(rows) != len(planes):
        raise ValueError("rows and planes differ in length")
    if not planes:
        return
    if len(planes) > MAX_PLANES:
        raise ValueError("more planes than EKV_MAX_PLANES in one call")
    device = require_cuda(dict(slot_map=slot_map))
    tokens = slot_map.shape[0] if slot_map.dim() == 1 else -1
    map_es = _vector(slot_map, "slot_map", None)
    first_row, first_plane = rows[0], planes[0]
    for row, plane in zip(rows, planes):
        require_cuda(dict(rows=row, planes=plane), device)
        if row.dim() < 2 or row.shape[0] != tokens or row.shape[1:] != plane.shape[1:]:
            raise ValueError("rows must be [tokens, ...] and planes [slots, ...] with the same row shape")
        if row.dtype != first_plane.dtype or plane.dtype != first_plane.dtype:
            raise TypeError("rows and planes must share one dtype (bitwise row copy)")
        if row.shape != first_row.shape or plane.shape != first_plane.shape:
            raise ValueError("all rows and all planes must share one shape")
    elements = first_row[0].numel() if tokens else 0
    if not tokens or not first_plane.shape[0] or not elements:
        return
    strides = {_row_stride(row, "rows") for row in rows}, {_row_stride(plane, "planes") for plane in planes}
    if len(strides[0]) != 1 or len(strides[1]) != 1:
        raise ValueError("rows and planes must each share one row stride")
    row_stride, plane_stride = strides[0].pop(), strides[1].pop()
    if plane_stride < elements:
        raise ValueError("plane rows overlap")
    itemsize = first_plane.element_size()
    call(
        "ekv_append_rows",
        u64_array(t.data_ptr() for t in rows), u64_array(t.data_ptr() for t in planes), len(planes),
        elements * itemsize, row_stride * itemsize, plane_stride * itemsize,
        slot_map.data_ptr(), map_es, tokens, first_plane.shape[0], device.index, stream_handle(device),
    )


__all__ = ["TableExtension", "extend_block_tables", "append_rows"]
