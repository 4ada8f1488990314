"""Attention of a batch whose requests share a prefix, the prefix read once for all.

The requests of a serving batch often begin with the same tokens (a system prompt, a
document many ask about), whose K and V rows one donor request keeps in the pool -- the
rows that ``shared_prefix.resolve_shared_block_locations`` finds.
``shared_prefix_attention`` attends over the paged planes directly: the shared tokens are
read once and multiplied with the query rows of every request together, each request's
own tokens are read through its own row of the block table, and the two parts join
through their log-sum-exp.  With ``shared_tokens=0`` it is paged attention.

``SharedPrefixAttention`` is the same bound to fixed tensors, for a decode loop or a
captured graph.  Nothing here has a counterpart in the reference, which leaves attention to
its engine.
"""

from __future__ import annotations

import ctypes as ct
import math

import torch

from ._lib import ATTENTION_MAX_ROW_TILES, call, index_esize, last_error, require_cuda, stream_handle, torch_binding
from .block_tables import _overlap, _vector

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}  # EKV_BF16, EKV_FP16
HEAD_DIMS = (64, 128)
# A positive number in 32 bits, whose product with log2(e) is finite there.
_LEAST_SCALE, _MOST_SCALE = 1.5e-45, 2.3e38


def _rows_ok(tensor: torch.Tensor, name: str) -> None:
    """[count, heads, dim] with contiguous, 16-byte aligned head rows."""
    if tensor.stride(2) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    step = 16 // tensor.element_size()
    if tensor.data_ptr() % 16 or any(s % step for n, s in zip(tensor.shape[:2], tensor.stride()[:2]) if n > 1):
        raise ValueError(f"{name} must have 16-byte aligned rows")


def _apart(shape, strides, width: int, name: str) -> None:
    """Entries of ``width`` elements that do not overlap, the heads of a token side by side or the tokens of a head."""
    (tokens, heads), (token, head) = shape, _strides_of(shape, strides)
    if (heads > 1 and head < width) or (tokens > 1 and token < width) or (
            tokens > 1 and heads > 1 and token < (heads - 1) * head + width and head < (tokens - 1) * token + width):
        raise ValueError(f"{name} rows overlap")


def _strides_of(shape, strides) -> tuple[int, int]:
    return tuple(s if n > 1 else 0 for n, s in zip(shape, strides))


def _strides(tensor: torch.Tensor) -> tuple[int, int]:
    """Strides of the first two dimensions; 0 for one of a single entry."""
    return _strides_of(tensor.shape[:2], tensor.stride()[:2])


def _collide(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors [tokens, heads] or [tokens, heads, dim] share an element.

    Exact for views of one buffer whose strides agree (slices of a fused projection, say); others count as sharing
    when their extents do.
    """
    if not _overlap(a, b):
        return False
    width_a, width_b = ((t.shape[2] if t.dim() == 3 else 1) * t.element_size() for t in (a, b))
    steps, counts = [], []
    for d in range(2):
        of_a, of_b = a.stride(d) * a.element_size(), b.stride(d) * b.element_size()
        if a.shape[d] > 1 and b.shape[d] > 1 and of_a != of_b:
            return True
        steps.append(of_a if a.shape[d] > 1 else of_b if b.shape[d] > 1 else 0)
        counts.append((a.shape[d], b.shape[d]))
    (large, of_large), (small, of_small) = sorted(zip(steps, counts), reverse=True)
    width = max(width_a, width_b)
    if max(of_small) > 1 and small < width or max(of_large) > 1 and large < (max(of_small) - 1) * small + width:
        return True
    # Rows of b lie at delta - i * large - j * small from those of a, with i and j differences of their indices.
    delta = b.data_ptr() - a.data_ptr()
    near = lambda x, step, of: [  # noqa: E731
        i for i in (range(x // step - 1, x // step + 3) if step else (0,)) if -of[1] < i < of[0]]
    return any(-width_b < delta - i * large - j * small < width_a
               for i in near(delta, large, of_large) for j in near(delta - i * large, small, of_small))


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and _strides(a) == _strides(b)


def _outputs(query, out, lse, return_lse):
    require_cuda(dict(query=query))
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if lse is None and return_lse:
        lse = torch.empty(query.shape[:2], dtype=torch.float32, device=query.device)
    return out, lse


def _bind(query, k_plane, v_plane, block_tables, lengths, page_size, shared_tokens, source_row, rows,
          query_starts, scale, out, lse):
    """Validated arguments of the C call up to the workspace, and the device."""
    device = require_cuda(dict(query=query, k_plane=k_plane, v_plane=v_plane, block_tables=block_tables,
                               lengths=lengths, rows=rows, query_starts=query_starts, out=out, lse=lse))
    if query.dim() != 3 or k_plane.dim() != 3 or v_plane.shape != k_plane.shape:
        raise ValueError("expected query [tokens, query_heads, dim] and planes [slots, kv_heads, dim]")
    if query.dtype not in _DTYPES:
        raise TypeError("query must be bfloat16 or float16")
    if k_plane.dtype != query.dtype or v_plane.dtype != query.dtype or out.dtype != query.dtype:
        raise TypeError("query, planes and out must share one dtype")
    tokens, query_heads, dim = query.shape
    slots, kv_heads, _ = k_plane.shape
    if dim not in HEAD_DIMS or k_plane.shape[2] != dim:
        raise ValueError("head dimension must be 64 or 128, the same in query and planes")
    if not kv_heads or not query_heads or query_heads % kv_heads:
        raise ValueError("query heads must be a positive multiple of KV heads")
    if out.shape != query.shape:
        raise ValueError("out must have query's shape")
    for tensor, name in ((query, "query"), (k_plane, "k_plane"), (v_plane, "v_plane"), (out, "out")):
        _rows_ok(tensor, name)
    for tensor, name in ((k_plane, "k_plane"), (v_plane, "v_plane"), (out, "out")):
        if any(n > 1 and s < dim for n, s in zip(tensor.shape[:2], tensor.stride()[:2])):
            raise ValueError(f"{name} rows overlap")
    _apart(out.shape[:2], out.stride()[:2], dim, "out")
    if lse is not None:
        if lse.dtype != torch.float32:
            raise TypeError("lse must be a float32 tensor")
        if lse.shape != (tokens, query_heads):
            raise ValueError("lse must be [tokens, query_heads]")
        _apart(lse.shape, lse.stride(), 1, "lse")
    outputs = [(out, "out")] if lse is None else [(out, "out"), (lse, "lse")]
    for tensor, name in outputs:
        if tensor is out and _same(out, query):
            pass
        elif _collide(tensor, query):
            raise ValueError(f"{name} overlaps query" + (" (it may be query itself)" if tensor is out else ""))
        if _collide(tensor, k_plane) or _collide(tensor, v_plane):
            raise ValueError(f"{name} overlaps a plane")
        if any(t is not None and _overlap(tensor, t) for t in (block_tables, lengths, rows, query_starts)):
            raise ValueError(f"{name} overlaps an index tensor")
    if lse is not None and _collide(out, lse):
        raise ValueError("out and lse overlap")
    if type(page_size) is not int or not 1 <= page_size < 1 << 31:
        raise ValueError("page_size outside the supported range")
    if block_tables.dim() != 2 or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be [rows, width] with contiguous rows")
    table_es = index_esize(block_tables, "block_tables")
    table_rows, table_width = block_tables.shape
    if table_width * page_size > (1 << 31) - 256:
        raise ValueError("a table row covers more than 2^31 - 256 positions")
    if type(shared_tokens) is not int or not 0 <= shared_tokens <= table_width * page_size:
        raise ValueError("shared_tokens outside the table's positions")
    if type(source_row) is not int or (shared_tokens and not 0 <= source_row < table_rows):
        raise ValueError("source row is outside the block table")
    batch = lengths.shape[0] if lengths.dim() == 1 else -1
    len_es = _vector(lengths, "lengths", None)
    rows_es = 8 if rows is None else _vector(rows, "rows", batch)
    starts_es = 8 if query_starts is None else _vector(query_starts, "query_starts", batch + 1)
    if query_starts is None and tokens != batch:
        raise ValueError("without query_starts every request has one query token")
    if batch + -(-tokens * query_heads // kv_heads // 256) > ATTENTION_MAX_ROW_TILES:
        raise ValueError("more requests and query tokens than one call takes")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not _LEAST_SCALE <= scale <= _MOST_SCALE:
        raise ValueError("scale must lie in [1.5e-45, 2.3e38]")
    return (
        query.data_ptr(), *_strides(query), k_plane.data_ptr(), *_strides(k_plane),
        v_plane.data_ptr(), *_strides(v_plane), slots,
        _DTYPES[query.dtype], dim, query_heads, kv_heads, tokens, batch,
        block_tables.data_ptr(), table_es, table_rows, table_width, block_tables.stride(0), page_size,
        None if rows is None else rows.data_ptr(), rows_es, lengths.data_ptr(), len_es,
        None if query_starts is None else query_starts.data_ptr(), starts_es, shared_tokens, source_row, scale,
        out.data_ptr(), *_strides(out),
        None if lse is None else lse.data_ptr(), *((0, 0) if lse is None else lse.stride()),
    ), device


def _workspace_bytes(query, kv_heads, batch, device) -> int:
    need = ct.c_int64()
    call("ekv_shared_prefix_workspace", query.shape[0], batch, query.shape[1], kv_heads, query.shape[2],
         device.index, ct.byref(need))
    return need.value


def shared_prefix_attention(query: torch.Tensor, k_plane: torch.Tensor, v_plane: torch.Tensor,
                            block_tables: torch.Tensor, lengths: torch.Tensor, *, page_size: int,
                            shared_tokens: int = 0, source_row: int = 0, rows: torch.Tensor | None = None,
                            query_starts: torch.Tensor | None = None, scale: float | None = None,
                            out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                            return_lse: bool = False):
    """Softmax attention of every query token over its request's tokens; returns ``out``
    (or ``(out, lse)`` when ``lse`` is given or ``return_lse`` is set).

    ``query`` [tokens, query_heads, dim] and the planes [slots, kv_heads, dim] are bfloat16 or
    float16 with ``dim`` 64 or 128; ``query_heads`` is a multiple of ``kv_heads`` (head h reads KV
    head ``h * kv_heads // query_heads``).  Tokens and heads may be strided, rows of ``dim``
    are contiguous and 16-byte aligned.

    ``lengths`` [requests] counts each request's tokens, its new ones included.  Without
    ``query_starts`` request b has the one new token ``query[b]``; with it (int32 / int64
    [requests + 1], ascending) its new tokens are ``query[query_starts[b]:query_starts[b + 1]]``,
    the last of the request, and each sees the tokens up to itself.  Query tokens of no
    request are left as they were in ``out`` and ``lse`` (uninitialised in tensors that the call makes).  ``out`` may be ``query`` itself; otherwise the outputs
    share no memory with the inputs or one another (interleaved views of one buffer are fine).

    Position t of request b is in slot ``page * page_size + t % page_size`` with ``page =
    block_tables[row, t // page_size]``, where ``row`` is ``source_row`` for the first
    ``shared_tokens`` positions and ``rows[b]`` (default b) behind them (where the shared positions end
    inside a page, the request's own entry for that page is read from there on).  A position without a
    slot (a negative page, one outside the planes, past the table) is skipped.  A query token
    that sees no position gets zeros and a log-sum-exp of minus infinity (one whose scores are all
    minus infinity NaN and minus infinity, as 0 / 0 and log 0 are).  Infinities and NaN
    reach the query tokens that see their position, no others.

    A table row covers up to 2^31 - 256 positions.  One call takes up to
    ``ATTENTION_MAX_ROW_TILES`` (1536) row tiles: one per request and one per 256 query rows of a
    KV head.  ``scale`` (1.5e-45 to 2.3e38) defaults to ``1 / sqrt(dim)``; ``lse`` is float32 [tokens, query_heads],
    the natural logarithm of the sum of the exponentials.  Scores, maxima, sums and outputs are
    held in 32 bits.  The weights are rounded to the inputs' type before they multiply V (half a step, up to 2^-8
    of each in bfloat16 and 2^-11 in float16, which also loses what is below 2^-32 of the largest); their sum
    is of the unrounded ones, and the result is rounded once more.  Sums are of weights up to 2^8 (2^15 in
    float16) times V, so a V above 2^100 may overflow them.  For serving: no gradients flow through it.
    """
    fast = torch_binding() if all(type(x) is int for x in (page_size, shared_tokens, source_row)) else None
    if fast is not None:
        try:
            rc, result, sums = fast.shared_prefix_attention(query, k_plane, v_plane, block_tables, lengths, page_size,
                                                            shared_tokens, source_row, rows, query_starts, scale, out, lse,
                                                            return_lse)
        except TypeError:  # not tensors: the checked path below reports it
            rc = fast.NOT_HANDLED
        if rc == 0:
            return result if sums is None else (result, sums)
        if rc == fast.KERNEL_ERROR:
            raise last_error("ekv_shared_prefix_attention")
    out, lse = _outputs(query, out, lse, return_lse)
    args, device = _bind(query, k_plane, v_plane, block_tables, lengths, page_size, shared_tokens, source_row, rows,
                         query_starts, scale, out, lse)
    need = _workspace_bytes(query, k_plane.shape[1], lengths.shape[0], device)
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    call("ekv_shared_prefix_attention", *args, workspace.data_ptr(), need, device.index, stream_handle(device))
    return out if lse is None else (out, lse)


class SharedPrefixAttention:
    """``shared_prefix_attention`` bound to fixed tensors for a hot loop (or a CUDA graph).

    Each call only launches; the tensors must outlive the object and keep their storage.
    The results are in ``out`` and ``lse`` (None unless given or asked for).  The object owns its
    workspace, so its calls must not overlap one another: two graphs that capture the same
    object must not replay at the same time.  The object must outlive the graphs that capture it.
    """

    def __init__(self, query, k_plane, v_plane, block_tables, lengths, *, page_size, shared_tokens=0, source_row=0,
                 rows=None, query_starts=None, scale=None, out=None, lse=None, return_lse=False):
        out, lse = _outputs(query, out, lse, return_lse)
        args, self.device = _bind(query, k_plane, v_plane, block_tables, lengths, page_size, shared_tokens,
                                  source_row, rows, query_starts, scale, out, lse)
        need = _workspace_bytes(query, k_plane.shape[1], lengths.shape[0], self.device)
        self.workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        self.out, self.lse = out, lse
        self._keep = (query, k_plane, v_plane, block_tables, lengths, rows, query_starts)
        self._args = (*args, self.workspace.data_ptr(), need, self.device.index)

    def __call__(self, stream: int | None = None) -> None:
        call("ekv_shared_prefix_attention", *self._args, stream_handle(self.device) if stream is None else stream)


__all__ = ["HEAD_DIMS", "SharedPrefixAttention", "shared_prefix_attention"]
