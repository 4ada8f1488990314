"""The serving operators of this package as they are measured: block tables, row append, shared-prefix attention.

Each case is one call of a decode or prompt step over a paged KV pool: ``extend_block_tables`` gives the
step's new tokens their slots, ``append_rows`` writes their K and V rows there, and
``shared_prefix_attention`` attends over a batch whose requests share a prefix.  ``own`` selects the
package's calls; otherwise the same results come from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEVICE = "cuda"
_LARGEST_FLOPS = 2.7e11
_LARGEST_BYTES = 1.2e9


# ------------------------------------------------------------------------------- cases

def listed():
    return [
        # One decode step of eight requests at page size 1, the pool layout of the repository's configurations.
        dict(name="tables decode 8", op="tables", requests=8, page=1, width=16384, held=12000, new_low=1, new_high=1,
             padding=0),
        # A large decode batch with pages of 16: most requests stay inside their last page.
        dict(name="tables decode 1024", op="tables", requests=1024, page=16, width=2048, held=20000, new_low=1,
             new_high=1, padding=64),
        # A step of prompts: ragged lengths, 64 requests, page size 1, so each token takes a page.
        dict(name="tables prompts", op="tables", requests=64, page=1, width=16384, held=4000, new_low=17,
             new_high=8000, padding=1000),
        # One layer's K and V of a 64-request decode step: 2 KiB rows (8 heads x 128).
        dict(name="append decode 64", op="append", tokens=64, heads=8, query_heads=32, dim=128, slots=65536,
             skip_every=0, dtype="bf16"),
        # One layer's K and V of a prompt step: 65,536 tokens, views of a fused projection, some skipped.
        dict(name="append prompts", op="append", tokens=65536, heads=8, query_heads=32, dim=128, slots=131072,
             skip_every=97, dtype="bf16"),
        # A tensor-parallel shard with one KV head, four requests, a short system prompt: latency.
        dict(name="attend 4 x 512", op="attend", requests=4, new_low=1, new_high=1, heads=1, group=4, dim=128,
             shared=512, own_low=1, own_high=60, page=1, dtype="bf16"),
        # The repository's 64-request batch with 8 KV heads x 128 (32 query heads), a 4,096-token prefix.
        dict(name="attend 64 x 4096", op="attend", requests=64, new_low=1, new_high=1, heads=8, group=4, dim=128,
             shared=4096, own_low=1, own_high=1000, page=1, dtype="bf16"),
        # A larger batch of long own contexts in fp16, pages of 16, eight query heads a KV head.
        dict(name="attend 128 x 16384", op="attend", requests=128, new_low=1, new_high=1, heads=8, group=8, dim=128,
             shared=16384, own_low=16, own_high=2000, page=16, dtype="fp16"),
        # A shared context of 131,072 tokens (a long document many requests ask about), short own parts.
        dict(name="attend 32 x 131072", op="attend", requests=32, new_low=1, new_high=1, heads=8, group=4, dim=128,
             shared=131072, own_low=5, own_high=500, page=64, dtype="bf16"),
        # The largest: 256 requests with 64 query heads over a 32,768-token prefix, pages of 128.
        dict(name="attend 256 x 32768", op="attend", requests=256, new_low=1, new_high=1, heads=8, group=8, dim=128,
             shared=32768, own_low=1, own_high=900, page=128, dtype="bf16"),
        # Drafts checked in one step: five tokens a request, causal among themselves, heads of 64, odd prefix.
        dict(name="attend drafts 48 x 5001", op="attend", requests=48, new_low=5, new_high=5, heads=8, group=3, dim=64,
             shared=5001, own_low=5, own_high=700, page=16, dtype="bf16"),
        # Prompts that continue a shared prefix: ragged chunks of new tokens, causal, odd prefix length.
        dict(name="attend prompts 8 x 8001", op="attend", requests=8, new_low=3, new_high=400, heads=8, group=4,
             dim=128, shared=8001, own_low=400, own_high=1200, page=16, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend", "attend"])
    if op == "tables":
        page = rng.choice([1, 16, 64])
        requests = _log_int(rng, 1, 1024)
        high = _log_int(rng, 1, min(8000, max(1, 260000 // requests)))
        held = rng.randrange(0, 24000)
        return dict(op=op, requests=requests, page=page, width=-(-(held + high) // page) + rng.randrange(1, 64),
                    held=held, new_low=rng.randint(1, high), new_high=high, padding=rng.randrange(0, 300))
    if op == "append":
        tokens = _log_int(rng, 1, 65536)
        heads = rng.choice([1, 2, 4, 8])
        return dict(op=op, tokens=tokens, heads=heads, query_heads=heads * rng.choice([1, 4, 8]),
                    dim=rng.choice([64, 128]), slots=tokens + rng.randrange(1, 65536),
                    skip_every=rng.choice([0, 13, 200]), dtype=rng.choice(["bf16", "fp16"]))
    while True:
        requests = _log_int(rng, 1, 256)
        several = rng.random() < 0.35
        high = _log_int(rng, 2, max(2, 1600 // requests)) if several else 1
        case = dict(op=op, requests=requests, new_low=rng.randint(1, high), new_high=high,
                    heads=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 2, 3, 4, 8]), dim=rng.choice([64, 128, 128]),
                    shared=_log_int(rng, 16, 65536), page=rng.choice([1, 16, 64, 128]),
                    dtype=rng.choice(["bf16", "fp16"]))
        case["own_low"] = high + rng.randrange(0, 64)
        case["own_high"] = case["own_low"] + _log_int(rng, 1, 2000)
        cost = work(case)
        if cost["flops"] <= _LARGEST_FLOPS and cost["bytes"] <= _LARGEST_BYTES:
            return case


def _ragged(count, low, high, step):
    """``count`` whole numbers spread over [low, high] in a fixed, unsorted order."""
    if count == 1:
        return [high]
    return [low + (high - low) * ((i * step) % count) // (count - 1) for i in range(count)]


def _step(count):
    """A step through ``count`` places that visits each of them."""
    return next(s for s in (7, 11, 13, 17, 19, 23, 29) if math.gcd(s, count) == 1)


def _new_tokens(case):
    return _ragged(case["requests"], case["new_low"], case["new_high"], _step(case["requests"]))


def _held(case):
    return _ragged(case["requests"], case["held"] // 2, case["held"], 1)


def _own_lengths(case):
    """Tokens of each request behind the shared prefix, its new ones among them."""
    own_tokens = _ragged(case["requests"], case["own_low"], case["own_high"], _step(case["requests"]))
    return [max(s, n) for s, n in zip(own_tokens, _new_tokens(case))]


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["op"] == "tables":
        taken = sum(_pages(held + new, case["page"]) - _pages(held, case["page"])
                    for held, new in zip(_held(case), _new_tokens(case)))
        tokens = sum(_new_tokens(case)) + case["padding"]
        # lengths, new tokens and rows in; starts and lengths out; pages in and out; slot and position of each token.
        return dict(bytes=20 * case["requests"] + 8 * taken + 8 * tokens, flops=2 * tokens)
    if case["op"] == "append":
        row = case["heads"] * case["dim"] * 2
        return dict(bytes=case["tokens"] * (2 * 2 * row + 4), flops=0)
    new, held = _new_tokens(case), _own_lengths(case)
    heads, dim, shared = case["heads"], case["dim"], case["shared"]
    query_heads = heads * case["group"]
    seen = sum(n * shared + n * s - n * (n - 1) // 2 for n, s in zip(new, held))
    rows = 2 * heads * dim * 2
    return dict(bytes=(shared + sum(held)) * (rows + 4.0 / case["page"]) + sum(new) * query_heads * (4 * dim + 4),
                flops=4 * dim * query_heads * seen)


# ------------------------------------------------------------------------------- inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(int(seed))

    def normal(*shape, dtype):
        return torch.randn(shape, generator=gen, device=_DEVICE, dtype=dtype)

    def shuffled(count):
        return torch.randperm(count, generator=gen, device=_DEVICE, dtype=torch.int32)

    state = dict(case=dict(case))
    if case["op"] == "tables":
        requests, page, width = case["requests"], case["page"], case["width"]
        held, new = _held(case), _new_tokens(case)
        taken = sum(_pages(h + n, page) - _pages(h, page) for h, n in zip(held, new))
        pages = shuffled(requests * width + taken + 7)
        state.update(block_tables=pages[:requests * width].reshape(requests, width).clone(),
                     free_pages=pages[requests * width:].clone(), lengths=_ints(held), new_tokens=_ints(new),
                     rows=shuffled(requests), max_tokens=sum(new) + case["padding"])
        return state
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "append":
        tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
        fused = normal(tokens, case["query_heads"] + 2 * heads, dim, dtype=dtype)
        k_rows, v_rows = fused[:, case["query_heads"]:].split(heads, dim=1)
        slot_map = shuffled(case["slots"])[:tokens].clone()
        if case["skip_every"]:
            slot_map[::case["skip_every"]] = -1
        state.update(rows=[k_rows, v_rows], slot_map=slot_map,
                     planes=[normal(case["slots"], heads, dim, dtype=dtype) for _ in range(2)])
        return state
    page, shared, heads, dim = case["page"], case["shared"], case["heads"], case["dim"]
    new, held = _new_tokens(case), _own_lengths(case)
    # Shared whole pages are the source's; each request owns the pages from the first partial one on.
    first = shared // page
    total = [_pages(shared + s, page) for s in held]
    width = max(total)
    pages = shuffled(first + sum(t - first for t in total) + 3)
    block_tables = torch.full((case["requests"], width), -1, dtype=torch.int32, device=_DEVICE)
    block_tables[:, :first] = pages[:first]
    cells = torch.arange(width, device=_DEVICE)[None, :]
    mine = (cells >= first) & (cells < _ints(total)[:, None])
    block_tables[mine] = pages[first:first + sum(t - first for t in total)]
    slots = pages.numel() * page
    k_plane, v_plane = (normal(slots, heads, dim, dtype=dtype) for _ in range(2))
    partial = shared - first * page
    if partial:  # the tokens of a partly shared page, in each request's copy of that page
        source = block_tables[0, first].long() * page + torch.arange(partial, device=_DEVICE)
        copies = block_tables[1:, first].long()[:, None] * page + torch.arange(partial, device=_DEVICE)
        for plane in (k_plane, v_plane):
            plane[copies] = plane[source]
    starts = torch.zeros(case["requests"] + 1, dtype=torch.int32, device=_DEVICE)
    starts[1:] = torch.cumsum(_ints(new), 0)
    # Queries a little sharper than unit normal, as trained attention is sharper than uniform.
    query = normal(sum(new), heads * case["group"], dim, dtype=dtype) * 1.5
    state.update(query=query, k_plane=k_plane, v_plane=v_plane, block_tables=block_tables,
                 lengths=_ints([shared + s for s in held]), query_starts=None if max(new) == 1 else starts,
                 out=torch.zeros_like(query), lse=torch.zeros(query.shape[:2], device=_DEVICE), most_own=max(held),
                 most_new=max(new))
    return state


# ------------------------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if own:
        return {"tables": _own_tables, "append": _own_append, "attend": _own_attend}[case["op"]](state)
    return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[case["op"]](state)


def _package():
    import sys
    from pathlib import Path

    root = str(Path(__file__).resolve().parents[1] / "elastic-kv-vmm_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


def _own_tables(state):
    if "call" not in state:
        _package()
        from ekv_b200.block_tables import extend_block_tables

        state["call"] = extend_block_tables
    step = state["call"](state["block_tables"], state["lengths"], state["new_tokens"], state["free_pages"],
                         page_size=state["case"]["page"], max_tokens=state["max_tokens"], rows=state["rows"])
    return dict(block_tables=state["block_tables"], query_starts=step.query_starts, slot_map=step.slot_map,
                positions=step.positions, lengths=step.lengths, pages_used=step.pages_used)


def _own_append(state):
    if "call" not in state:
        _package()
        from ekv_b200.block_tables import append_rows

        state["call"] = append_rows
    state["call"](state["rows"], state["slot_map"], state["planes"])
    return dict(planes=state["planes"])


def _own_attend(state):
    if "call" not in state:
        _package()
        from ekv_b200.prefix_attention import shared_prefix_attention

        state["call"] = shared_prefix_attention
    case = state["case"]
    state["call"](state["query"], state["k_plane"], state["v_plane"], state["block_tables"], state["lengths"],
                  page_size=case["page"], shared_tokens=case["shared"], query_starts=state["query_starts"],
                  out=state["out"], lse=state["lse"])
    return dict(out=state["out"], lse=state["lse"])


def _plain_tables(state):
    page, tables, rows = state["case"]["page"], state["block_tables"], state["rows"].long()
    held, new, free = state["lengths"].long(), state["new_tokens"].long(), state["free_pages"]
    capacity = state["max_tokens"]
    had = (held + page - 1) // page
    active = (new > 0) & (held + new <= tables.shape[1] * page)
    need = torch.where(active, (held + new + page - 1) // page - had, 0)
    tokens = torch.where(active, new, 0)
    taken = torch.cumsum(need, 0)
    fits = (taken <= free.numel()) & (torch.cumsum(tokens, 0) <= capacity)
    need, tokens = torch.where(fits, need, 0), torch.where(fits, tokens, 0)
    ends, taken = torch.cumsum(tokens, 0), torch.cumsum(need, 0)
    column = torch.arange(tables.shape[1], device=tables.device)[None, :] - had[:, None]
    place = torch.clamp(column + (taken - need)[:, None], 0, free.numel() - 1)
    tables[rows] = torch.where((column >= 0) & (column < need[:, None]), free[place], tables[rows])
    token = torch.arange(capacity, device=tables.device)
    request = torch.clamp(torch.searchsorted(ends, token, right=True), max=held.numel() - 1)
    position = held[request] + token - (ends - tokens)[request]
    inside = token < ends[-1]
    at = torch.clamp(position // page, 0, tables.shape[1] - 1)
    slot = tables[rows[request], at].long() * page + position % page
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    return dict(block_tables=tables, query_starts=starts.int(), slot_map=torch.where(inside, slot, -1).int(),
                positions=torch.where(inside, position, -1).int(), lengths=(held + tokens).int(),
                pages_used=taken[-1:].int())


def _plain_append(state):
    slot_map = state["slot_map"].long()
    keep = slot_map >= 0
    state["planes"][0][slot_map[keep]] = state["rows"][0][keep]
    state["planes"][1][slot_map[keep]] = state["rows"][1][keep]
    return dict(planes=state["planes"])


def _plain_attend(state):
    case, tables, lengths = state["case"], state["block_tables"].long(), state["lengths"].long()
    page, shared, heads, group, dim = case["page"], case["shared"], case["heads"], case["group"], case["dim"]
    k_plane, v_plane, query = state["k_plane"], state["v_plane"], state["query"]
    count, most_own, most_new = query.shape[0], state["most_own"], state["most_new"]
    device = query.device
    rows = query.float().reshape(count, heads, group, dim) * (1.0 / math.sqrt(dim))
    starts = state["query_starts"]
    starts = torch.arange(count + 1, device=device) if starts is None else starts.long()
    token = torch.arange(count, device=device)
    request = torch.searchsorted(starts[1:], token, right=True)
    at = token - starts[request]
    seen = lengths[request] - (starts[request + 1] - starts[request]) + at + 1
    # The shared tokens, through the source's table, for every row at once.
    position = torch.arange(shared, device=device)
    slot = tables[0, position // page] * page + position % page
    k_shared, v_shared = k_plane[slot].float(), v_plane[slot].float()
    first = torch.matmul(rows.permute(1, 0, 2, 3).reshape(heads, count * group, dim), k_shared.permute(1, 2, 0))
    first = first.reshape(heads, count, group, shared).permute(1, 0, 2, 3)
    # Each request's own tokens, padded to the longest.
    position = shared + torch.arange(most_own, device=device)[None, :]
    cell = torch.clamp(position // page, max=tables.shape[1] - 1).expand(lengths.numel(), -1)
    page_of = torch.clamp(tables.gather(1, cell), min=0)
    there = position < lengths[:, None]
    slot = page_of * page + position % page
    k_own = torch.where(there[..., None, None], k_plane[slot].float(), 0.0)
    v_own = torch.where(there[..., None, None], v_plane[slot].float(), 0.0)
    padded = torch.zeros((lengths.numel(), most_new, heads, group, dim), device=device)
    padded[request, at] = rows
    padded = padded.permute(0, 2, 1, 3, 4).reshape(-1, heads, most_new * group, dim)
    second = torch.matmul(padded, k_own.permute(0, 2, 3, 1)).reshape(-1, heads, most_new, group, most_own)
    second = second[request, :, at]
    visible = (position < seen[:, None])[:, None, None, :]
    second = torch.where(visible, second, -math.inf)
    top = torch.maximum(first.amax(-1, keepdim=True), second.amax(-1, keepdim=True))
    first, second = torch.exp(first - top), torch.exp(second - top)
    total = first.sum(-1, keepdim=True) + second.sum(-1, keepdim=True)
    out = torch.matmul(first.permute(1, 0, 2, 3).reshape(heads, count * group, shared), v_shared.permute(1, 0, 2))
    out = out.reshape(heads, count, group, dim).permute(1, 0, 2, 3)
    padded = torch.zeros((lengths.numel(), most_new, heads, group, most_own), device=device)
    padded[request, at] = second
    padded = padded.permute(0, 2, 1, 3, 4).reshape(-1, heads, most_new * group, most_own)
    own_part = torch.matmul(padded, v_own.permute(0, 2, 1, 3)).reshape(-1, heads, most_new, group, dim)[request, :, at]
    out = (out + own_part) / total
    lse = (top + torch.log(total)).squeeze(-1)
    state["out"].copy_(out.reshape(query.shape).to(query.dtype))
    state["lse"].copy_(lse.reshape(query.shape[:2]))
    return dict(out=state["out"], lse=state["lse"])


# ------------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    state = prepare(case, seed)
    if case["op"] == "append":
        result = [plane.double() for plane in state["planes"]]
        for plane, rows in zip(result, state["rows"]):
            # A skipped token falls on an extra row behind the plane, which is dropped again.
            wide = torch.cat([plane, plane.new_zeros(1, *plane.shape[1:])])
            target = torch.where(state["slot_map"] < 0, case["slots"], state["slot_map"])
            wide.index_copy_(0, target.long(), rows.double())
            plane.copy_(wide[:-1])
        return dict(planes=result)
    page, heads, group, dim = case["page"], case["heads"], case["group"], case["dim"]
    query = state["query"].double()
    out, lse = torch.zeros_like(query), torch.zeros(query.shape[:2], dtype=torch.float64, device=query.device)
    begin = 0
    for b, (new, held) in enumerate(zip(_new_tokens(case), _own_lengths(case))):
        length = case["shared"] + held
        position = torch.arange(length, device=query.device)
        slot = state["block_tables"][b].long().repeat_interleave(page)[:length] * page + position % page
        keys, values = state["k_plane"][slot].double(), state["v_plane"][slot].double()
        rows = query[begin:begin + new].reshape(new, heads, group, dim)
        scores = torch.einsum("nhgd,thd->nhgt", rows, keys) / math.sqrt(dim)
        hidden = position[None, :] > (length - new + torch.arange(new, device=query.device))[:, None]
        scores = scores.masked_fill(hidden[:, None, None, :], -math.inf)
        out[begin:begin + new] = torch.einsum("nhgt,thd->nhgd", torch.softmax(scores, -1), values).reshape(new, -1, dim)
        lse[begin:begin + new] = torch.logsumexp(scores, -1).reshape(new, -1)
        begin += new
    return dict(out=out, lse=lse)
