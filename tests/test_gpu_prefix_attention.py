"""Shared-prefix attention on the device against the 64-bit CPU restatement.

Tolerance.  The kernel multiplies exact products of 16-bit inputs in 32 bits; the weights
p_j = exp(s_j - m) may be rounded once to the 16-bit type (half a step, u = eps / 2, of p_j)
before the product with V, and the result once to the type.  With A = sum_j p_j |v_j| /
sum_j p_j that is u (A + |o|).  In 32 bits (e = 2^-24): a score has at most (dim + 4) e reach
of error, which moves p_j, sum p and so o by twice that times A; sums of n terms add n e each
(numerator and denominator), the exponential 4 e.  fp16 weights below 2^-14 round by 2^-25 of the
largest weight instead: n 2^-25 max|v|.  The log-sum-exp has the same terms without u, plus
4 e of its own value.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block_tables as obt
from oracle import prefix_attention as opa

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
MARK = 7.0  # in rows that a call must leave alone


def _np(tensor):
    return tensor.detach().double().cpu().numpy()


class Case:
    """A pool of shuffled pages, tables that share their first pages, and ragged lengths (all on the host)."""

    def __init__(self, *, lengths, shared, page=16, heads=2, group=4, dim=128, dtype=torch.bfloat16, new=None,
                 seed=0, spread=1.5, spare_width=1, index=torch.int32, tail=0):
        gen = torch.Generator().manual_seed(seed)
        batch = len(lengths)
        self.page, self.shared, self.dtype = page, shared, dtype
        self.lengths = torch.tensor(lengths, dtype=index).reshape(batch)
        new_list = [1] * batch if new is None else list(new)
        self.starts = None if new is None else torch.tensor(np.concatenate([[0], np.cumsum(new_list)]), dtype=index)
        first = shared // page
        need = [max(0, -(-length // page) - first) for length in lengths]
        width = max([first + n for n in need] + [-(-shared // page), 1]) + spare_width
        total = first + sum(need) + 2 + (1 if shared % page else 0)
        pages = torch.randperm(total, generator=gen)
        self.tables = torch.full((batch + 1, width), -1, dtype=index)
        self.tables[:, :first] = pages[:first]
        at = first
        self.source = batch  # the donor has a row of its own, behind the batch's
        if shared % page:
            self.tables[batch, first] = pages[at]
            at += 1
        for b, n in enumerate(need):
            self.tables[b, first:first + n] = pages[at:at + n].to(index)
            at += n
        self.k, self.v = (torch.randn((total * page, heads, dim), generator=gen).to(dtype) for _ in range(2))
        tokens = sum(new_list) + tail
        self.query = (torch.randn((tokens, heads * group, dim), generator=gen) * spread).to(dtype)

    def want(self, **change):
        args = dict(page_size=self.page, shared_tokens=self.shared, source_row=self.source,
                    query_starts=None if self.starts is None else self.starts.numpy())
        args.update(change)
        return opa.attend(_np(self.query), _np(self.k), _np(self.v), self.tables.numpy(), self.lengths.numpy(), **args)

    def run(self, device, **change):
        from ekv_b200.prefix_attention import shared_prefix_attention

        args = dict(page_size=self.page, shared_tokens=self.shared, source_row=self.source,
                    query_starts=None if self.starts is None else self.starts.to(device),
                    out=torch.full_like(self.query, MARK, device=device),
                    lse=torch.full(self.query.shape[:2], MARK, device=device))
        args.update(change)
        return shared_prefix_attention(self.query.to(device), self.k.to(device), self.v.to(device),
                                       self.tables.to(device), self.lengths.to(device), **args)


def compare(got, want, dtype, v_max, dim):
    out, lse = _np(got[0]), _np(got[1])
    expected, expected_lse, weight, reach, seen = want
    absent = np.isnan(expected).all((1, 2))
    assert (out[absent] == MARK).all() and (lse[absent] == MARK).all()
    out, lse, expected, expected_lse = out[~absent], lse[~absent], expected[~absent], expected_lse[~absent]
    weight, reach, seen = weight[~absent], reach[~absent], seen[~absent][:, None]
    u = torch.finfo(dtype).eps / 2
    inner = 2 * (dim + 4) * E * reach + (2 * seen + 8) * E
    small = seen * 2.0 ** -25 * v_max if dtype == torch.float16 else 0 * seen
    tolerance = u * (weight + np.abs(expected)) * (1 + 2 * u) + 2 * inner[..., None] * weight + small[..., None]
    excess = np.abs(out - expected) - tolerance
    assert not (excess > 0).any(), (excess.max(), np.argwhere(excess > 0)[:5], int((excess > 0).sum()))
    empty = np.isneginf(expected_lse)
    assert (np.isneginf(lse) == empty).all() and (out[empty] == 0).all()
    lse[empty] = expected_lse[empty] = 0.0
    assert not (np.abs(lse - expected_lse) > inner + 4 * E * np.abs(expected_lse)).any()


def check(case, device, **change):
    got = case.run(device, **change)
    compare(got, case.want(), case.dtype, float(case.v.double().abs().max()), case.query.shape[2])
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (1, 8), (2, 3), (8, 4), (3, 16)])
def test_decode(dtype, dim, heads, group, cuda_device):
    """Single tokens: a prefix that ends inside a page and a tile, ragged own parts."""
    check(Case(lengths=[301, 300, 417, 905, 302], shared=300, heads=heads, group=group, dim=dim, dtype=dtype),
          cuda_device)


@pytest.mark.parametrize("page", [1, 5, 16, 64, 128, 256])
@pytest.mark.parametrize("shared", [0, 1, 127, 128, 129, 640])
def test_page_sizes_and_prefix_lengths(page, shared, cuda_device):
    lengths = [shared + n for n in (1, 2, 63, 64, 65, 127, 128, 129, 260)]
    check(Case(lengths=lengths, shared=shared, page=page, heads=1, group=2, dim=64, index=torch.int64), cuda_device)


def test_short_and_empty_requests(cuda_device):
    """Lengths of zero, below, at and just above the prefix: rows that see part of it or nothing."""
    case = Case(lengths=[0, 1, 0, 5, 199, 200, 201, 0, 128, 129], shared=200, page=16)
    got = check(case, cuda_device)
    assert int(torch.isinf(got[1]).all(1).sum()) == 3
    check(Case(lengths=[0, 0], shared=0), cuda_device)
    check(Case(lengths=[0, 0, 0], shared=64), cuda_device)
    check(Case(lengths=[-5, 3], shared=2), cuda_device)


@pytest.mark.parametrize("requests", [1, 2, 33, 130, 300])
def test_batch_sizes(requests, cuda_device):
    lengths = [150 + (37 * b) % 210 for b in range(requests)]
    check(Case(lengths=lengths, shared=150, heads=2, group=2, dim=64, page=1), cuda_device)


@pytest.mark.parametrize("dtype,dim,group", [(torch.bfloat16, 128, 4), (torch.float16, 64, 1), (torch.bfloat16, 64, 7)])
def test_several_new_tokens(dtype, dim, group, cuda_device):
    """Ragged new tokens, causal among themselves; requests without any, more new tokens than
    length (the first ones see nothing or part of the prefix), and tokens behind the last request."""
    new = [1, 5, 0, 70, 130, 3, 0, 40]
    lengths = [131, 140, 200, 215, 260, 2, 0, 150]
    check(Case(lengths=lengths, new=new, shared=130, dtype=dtype, dim=dim, group=group, tail=6), cuda_device)


def test_prompts_without_a_prefix(cuda_device):
    """Whole prompts: every tile on the diagonal."""
    check(Case(lengths=[1, 127, 128, 129, 300], new=[1, 127, 128, 129, 300], shared=0, heads=1, group=2, dim=64),
          cuda_device)


def test_many_query_rows_over_a_prefix(cuda_device):
    """More query rows than one tile holds, several tiles of keys, both parts split."""
    check(Case(lengths=[2000 + 3 * b for b in range(80)], shared=1999, heads=1, group=8, dim=128), cuda_device)


def test_long_context(cuda_device):
    check(Case(lengths=[70001, 70500], shared=70000, heads=1, group=2, dim=64, page=64), cuda_device)
    check(Case(lengths=[40000, 3], shared=0, heads=1, group=2, dim=128, page=64), cuda_device)


def test_shared_and_own_reading_agree(cuda_device):
    """The same tokens read through the donor's row and through each request's own."""
    case = Case(lengths=[290, 256, 400], shared=256, page=16)
    one = case.run(cuda_device)
    two = case.run(cuda_device, shared_tokens=0)
    v_max = float(case.v.double().abs().max())
    compare(one, case.want(), case.dtype, v_max, 128)
    compare(two, case.want(), case.dtype, v_max, 128)


def test_positions_without_a_slot_are_skipped(cuda_device):
    """Negative pages, pages past the planes, a table narrower than the lengths, rows outside the table."""
    case = Case(lengths=[200, 210, 450, 333], shared=96, page=16, spare_width=0)
    case.tables[1, 9] = -1
    case.tables[2, 8] = 1 << 20
    case.tables[2, 7] = (1 << 31) - 1
    case.tables[case.source, 2] = -3
    case.lengths[3] = 5000
    check(case, cuda_device)
    rows = torch.tensor([2, -1, 99, 0])
    got = case.run(cuda_device, rows=rows.to(cuda_device))
    compare(got, case.want(rows=rows.numpy()), case.dtype, float(case.v.double().abs().max()), 128)


def test_nothing_behind_a_request_is_read(cuda_device):
    """NaN in every slot no request sees (the rest of its last page, unused pages), in K and in V."""
    case = Case(lengths=[150, 97, 130, 300], shared=90, page=16)
    want = case.want()
    used = np.zeros(case.k.shape[0], dtype=bool)
    for b, length in enumerate(case.lengths.tolist()):
        position = np.arange(length)
        slot = opa.slots_of(case.tables[b].numpy(), position, 16, len(used))
        donor = opa.slots_of(case.tables[case.source].numpy(), position, 16, len(used))
        used[np.where(position < 90, donor, slot)] = True
    assert not used.all()
    v_max = float(case.v.double().abs().max())
    for value in (float("nan"), float("inf"), torch.finfo(case.dtype).min):
        case.k[~torch.from_numpy(used)] = value
        case.v[~torch.from_numpy(used)] = value
        compare(case.run(cuda_device), want, case.dtype, v_max, 128)


@pytest.mark.parametrize("odd", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype,dim,shared,lengths,new,at", [
    # Requests of several new tokens (group 4), from tiles of 256 rows to fewer than 16, `at` a new token's place.
    (torch.bfloat16, 128, 40, [290, 100, 44], [200, 37, 2], [130, 61, 70, 90, 200, 289]),
    (torch.float16, 64, 0, [70, 9, 1], [70, 3, 1], [0, 7, 64, 65]),
    # Requests shorter than the prefix, few and many: `at` is a shared position that some see.
    (torch.bfloat16, 64, 500, [3, 130, 400, 520], None, [130, 400, 401, 499]),
    (torch.float16, 128, 300, [10 + 7 * i for i in range(48)], None, [9, 10, 200, 290]),
])
def test_infinities_and_nan_where_only_others_look(dtype, dim, shared, lengths, new, at, odd, cuda_device):
    """An odd V value reaches the rows that see its position and no others; an odd K value likewise."""
    case = Case(lengths=lengths, shared=shared, new=new, dtype=dtype, dim=dim)
    source = case.tables[case.source]

    def slot(request, position):
        row = source if position < shared else case.tables[request]
        return int(row[position // case.page]) * case.page + position % case.page

    for plane in (case.v, case.k):
        kept = plane.clone()
        for i, position in enumerate(at):
            if plane is case.k and position == 0:
                continue  # a row may see nothing else: 0 / 0 if its score is minus infinity
            for request in range(len(lengths)):
                if position < max(lengths[request], shared) and not (position < shared and request):
                    plane[slot(request, position), i % 2, 3 * i + 1] = odd
        got = case.run(cuda_device)
        with np.errstate(invalid="ignore"):
            want = case.want()
        plane.copy_(kept)
        out, lse = _np(got[0]), _np(got[1])
        bad = ~np.isfinite(want[0])
        assert bad.any() and not bad.all()
        assert (np.isfinite(out) == ~bad).all() and (np.isfinite(lse) == np.isfinite(want[1])).all()
        for values in (want[0], want[2], out):
            values[bad] = 0.0
        with np.errstate(invalid="ignore"):  # rows of an odd key have no tolerance to speak of
            compare((torch.from_numpy(out), torch.from_numpy(lse)), want, dtype, float(case.v.double().abs().max()), dim)


@pytest.mark.parametrize("dim,page", [(128, 1), (64, 1), (128, 16), (64, 3)])
def test_many_short_items(dim, page, cuda_device):
    """Requests of 17 to 72 new tokens between decoding ones: items of one to four tiles that take turns on the
    two halves of a block, among larger ones, with holes in the table (whose rows take the slower copy)."""
    gen = torch.Generator().manual_seed(9)
    new = [21, 5, 0, 1, 0, 5, 2, 1, 0, 2, 5, 0, 5, 1, 1, 25, 41, 72, 1, 1, 17, 12, 5, 44, 5, 62, 1, 17, 0, 1, 5, 1, 5, 64, 1, 1, 1, 30]
    own = torch.randint(0, 420, (len(new),), generator=gen).tolist()
    case = Case(lengths=[max(70 + n, w) for n, w in zip(own, new)], shared=70, page=page, heads=8, group=5, dim=dim, new=new)
    for holes in range(3):
        case.tables[torch.rand(case.tables.shape, generator=gen) < 0.1 * holes] = -1
        first = check(case, cuda_device)
        for _ in range(4):
            again = case.run(cuda_device)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_output_in_the_query(cuda_device):
    """`out` may be `query` itself, rows that are summed again included; lse transposed."""
    from ekv_b200.prefix_attention import shared_prefix_attention

    case = Case(lengths=[60, 20, 300], new=[50, 3, 1], shared=30, tail=4)
    slot = int(case.tables[0][50 // 16]) * 16 + 50 % 16
    case.v[slot, 1, 7] = float("nan")  # a new token of request 0, seen by its last ten
    apart = case.run(cuda_device)
    query = case.query.to(cuda_device)
    lse = torch.full((8, case.query.shape[0]), MARK, device=cuda_device).t()
    out, _ = shared_prefix_attention(query, *(t.to(cuda_device) for t in (case.k, case.v, case.tables, case.lengths)),
                                     page_size=16, shared_tokens=30, source_row=case.source, lse=lse,
                                     query_starts=case.starts.to(cuda_device), out=query)
    assert out.data_ptr() == query.data_ptr()
    assert int(torch.isnan(out[:54]).sum()) == 10 * 4 and torch.equal(out[54:].cpu(), case.query[54:])
    torch.testing.assert_close(out[:54], apart[0][:54], rtol=0, atol=0, equal_nan=True)
    assert torch.equal(lse, apart[1])


def test_more_query_heads_than_a_tile_has_rows(cuda_device):
    check(Case(lengths=[70, 200], new=[3, 1], shared=50, heads=1, group=300, dim=64), cuda_device)


def test_most_requests_of_one_call(cuda_device):
    """1530 requests and their six tiles of 256 query rows: as many as one call takes."""
    check(Case(lengths=[40 + b % 7 for b in range(1530)], shared=40, heads=1, group=1, dim=64), cuda_device)


def test_calls_captured_without_a_plan(cuda_device):
    """The function itself in two graphs of one pool, replayed in turn."""
    from ekv_b200.prefix_attention import shared_prefix_attention

    cases = [Case(lengths=[210 + 30 * b for b in range(6)], shared=200, seed=s) for s in (3, 4)]
    dev = [[t.to(cuda_device) for t in (c.query, c.k, c.v, c.tables, c.lengths)] for c in cases]

    def run(i):
        return shared_prefix_attention(*dev[i], page_size=16, shared_tokens=200, source_row=6, return_lse=True)

    run(0)
    graphs, results, pool = [], [], torch.cuda.graph_pool_handle()
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], pool=pool):
            results.append(run(i))
    for _ in range(2):
        for i, c in enumerate(cases):
            graphs[i].replay()
            compare(results[i], c.want(), c.dtype, float(c.v.double().abs().max()), 128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sharp_and_growing_scores(dtype, cuda_device):
    """Scores whose maximum grows along the tokens (rescaling at every tile) and nearly one-hot rows."""
    case = Case(lengths=[700, 900], shared=500, heads=1, group=2, dim=64, dtype=dtype, spread=0.5)
    slot = opa.slots_of(case.tables[1].numpy(), np.arange(900), 16, case.k.shape[0])
    donor = opa.slots_of(case.tables[case.source].numpy(), np.arange(500), 16, case.k.shape[0])
    ramp = torch.linspace(0.2, 6.0, 900)[:, None, None]
    slots = torch.from_numpy(np.concatenate([donor, slot[500:]]))
    case.k[slots] = (case.query[1, :1][None].float() * ramp).to(dtype)
    check(case, cuda_device)
    case.query = (case.query.float() * 40).to(dtype)
    check(case, cuda_device)


def test_scale_and_single_head_layouts(cuda_device):
    case = Case(lengths=[90, 133], shared=64, heads=1, group=1, dim=64)
    got = case.run(cuda_device, scale=0.5)
    compare(got, case.want(scale=0.5), case.dtype, float(case.v.double().abs().max()), 64)


def test_strided_tensors(cuda_device):
    """Queries out of a fused projection, K and V interleaved in one pool, strided out and lse."""
    from ekv_b200.prefix_attention import shared_prefix_attention

    case = Case(lengths=[290, 301, 350], shared=256, heads=2, group=4, dim=64, spare_width=3)
    tokens, query_heads, dim = case.query.shape
    fused = torch.full((tokens, query_heads + 4, dim), float("nan"), dtype=case.dtype, device=cuda_device)
    fused[:, :query_heads] = case.query.to(cuda_device)
    pool = torch.full((case.k.shape[0], 2, 2, dim + 8), float("nan"), dtype=case.dtype, device=cuda_device)
    pool[:, 0, :, :dim] = case.k.to(cuda_device)
    pool[:, 1, :, :dim] = case.v.to(cuda_device)
    tables = torch.full((4, case.tables.shape[1] + 5), -1, dtype=torch.int32, device=cuda_device)
    tables[:, :case.tables.shape[1]] = case.tables.to(cuda_device)
    out = torch.full((query_heads, tokens + 1, dim + 16), MARK, dtype=case.dtype, device=cuda_device)
    lse = torch.full((query_heads, tokens + 2), MARK, device=cuda_device)
    shared_prefix_attention(
        fused[:, :query_heads], pool[:, 0, :, :dim], pool[:, 1, :, :dim], tables[:, :case.tables.shape[1]],
        case.lengths.to(cuda_device), page_size=16, shared_tokens=256, source_row=3,
        out=out[:, :tokens, :dim].transpose(0, 1), lse=lse[:, :tokens].t())
    compare((out[:, :tokens, :dim].transpose(0, 1), lse[:, :tokens].t()), case.want(), case.dtype,
            float(case.v.double().abs().max()), dim)
    assert bool((out[:, tokens:] == MARK).all()) and bool((out[:, :, dim:] == MARK).all())
    assert bool((lse[:, tokens:] == MARK).all())


def test_slots_past_32_bit_offsets(cuda_device):
    """A plane of more than 2^31 elements, its rows in the first and the last slots."""
    from ekv_b200.prefix_attention import shared_prefix_attention

    case = Case(lengths=[70, 96], shared=64, page=16, heads=2, group=2, dim=128)
    pages, slots = case.k.shape[0] // 16, ((1 << 31) // 1024 + 4096) // 16 * 16
    pool = torch.empty((slots, 4, 2, 128), dtype=case.dtype, device=cuda_device)
    shift = torch.where(torch.arange(pages) % 2 == 1, slots // 16 - pages, 0)
    place = ((torch.arange(pages) + shift)[:, None] * 16 + torch.arange(16)).reshape(-1)
    pool[place.to(cuda_device), 1] = case.k.to(cuda_device)
    pool[place.to(cuda_device), 3] = case.v.to(cuda_device)
    tables = torch.where(case.tables >= 0, case.tables + shift[case.tables.clamp(min=0).long()].int(), -1)
    got = shared_prefix_attention(case.query.to(cuda_device), pool[:, 1], pool[:, 3], tables.to(cuda_device),
                                  case.lengths.to(cuda_device), page_size=16, shared_tokens=64, source_row=2,
                                  return_lse=True)
    compare(got, case.want(), case.dtype, float(case.v.double().abs().max()), 128)


def test_outputs_are_optional_and_repeat_bit_for_bit(cuda_device):
    case = Case(lengths=[600, 700, 800], shared=512, heads=2, group=8)
    out, lse = case.run(cuda_device)
    alone = case.run(cuda_device, out=None, lse=None)
    assert isinstance(alone, torch.Tensor) and torch.equal(alone, out)
    again = case.run(cuda_device, out=None, lse=None, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_empty_calls(cuda_device):
    from ekv_b200.prefix_attention import shared_prefix_attention

    planes = torch.zeros((8, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    tables = torch.zeros((1, 2), dtype=torch.int32, device=cuda_device)
    none = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    out = shared_prefix_attention(planes[:0], planes, planes, tables, none, page_size=4)
    assert out.shape == (0, 2, 64)
    out, lse = shared_prefix_attention(planes[:0], planes, planes, tables, none, page_size=4, return_lse=True,
                                       query_starts=torch.zeros(1, dtype=torch.int32, device=cuda_device))
    assert lse.shape == (0, 2)
    # Planes without slots: every position is skipped.
    out, lse = shared_prefix_attention(planes[:1], planes[:0], planes[:0], tables,
                                       torch.ones(1, dtype=torch.int32, device=cuda_device), page_size=4,
                                       shared_tokens=2, return_lse=True)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


def test_plan_captured_with_changing_lengths(cuda_device):
    """One plan, captured once; lengths and tables change between replays, on another stream."""
    from ekv_b200.prefix_attention import SharedPrefixAttention

    cases = [Case(lengths=ls, shared=200, page=16, seed=i, spare_width=60 - max(-(-n // 16) for n in ls))
             for i, ls in enumerate(([201, 300, 900], [700, 0, 200], [204, 205, 960]))]
    big = max(c.k.shape[0] for c in cases)
    k, v = (torch.zeros((big, 2, 128), dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    query, tables = cases[0].query.to(cuda_device), cases[0].tables.to(cuda_device)
    lengths = cases[0].lengths.to(cuda_device)
    plan = SharedPrefixAttention(query, k, v, tables, lengths, page_size=16, shared_tokens=200, source_row=3,
                                 return_lse=True)
    plan()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan()
    stream = torch.cuda.Stream()
    for case in cases:
        for tensor, host in ((query, case.query), (tables, case.tables), (lengths, case.lengths)):
            tensor.copy_(host)
        k[:case.k.shape[0]].copy_(case.k)
        v[:case.v.shape[0]].copy_(case.v)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.current_stream().wait_stream(stream)
        compare((plan.out, plan.lse), case.want(), case.dtype, float(case.v.double().abs().max()), 128)


def test_calls_on_two_streams_at_once(cuda_device):
    cases = [Case(lengths=[900 + 10 * b for b in range(20)], shared=800, heads=4, group=4, seed=s) for s in (1, 2)]
    dev = [[t.to(cuda_device) for t in (c.query, c.k, c.v, c.tables, c.lengths)] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    from ekv_b200.prefix_attention import shared_prefix_attention

    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(6):
        for i, (stream, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(stream):
                results[i].append(shared_prefix_attention(*dev[i], page_size=16, shared_tokens=800,
                                                          source_row=c.source, return_lse=True))
    torch.cuda.synchronize()
    for c, got in zip(cases, results):
        for out, lse in got[1:]:
            assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])
        compare(got[0], c.want(), c.dtype, float(c.v.double().abs().max()), 128)


def test_a_step_of_a_serving_loop(cuda_device):
    """Pages, append and attention together, as a step uses them, captured once and replayed: three
    steps of a batch that shares a prefix, each continuing what the one before wrote."""
    from ekv_b200.block_tables import append_rows, extend_block_tables
    from ekv_b200.prefix_attention import SharedPrefixAttention

    gen = torch.Generator().manual_seed(5)
    page, shared, batch, heads, group, dim, most = 16, 100, 3, 2, 4, 64, 60
    pages = torch.randperm(40, generator=gen).to(torch.int32)
    tables = torch.full((batch + 1, 24), -1, dtype=torch.int32)
    tables[:, :7] = pages[:7]  # six whole pages of the prefix and the donor's partial one
    tables[:batch, 6] = -1
    slots = 40 * page
    pool = torch.randn((slots, 2, heads, dim), generator=gen).bfloat16()
    donor = torch.from_numpy(opa.slots_of(tables[batch].numpy(), np.arange(shared), page, slots))
    # Each request starts with a page of its own for the four tokens of the partly shared page.
    tables[:batch, 6] = pages[7:10]
    free = pages[10:].clone()
    host_tables, lengths = tables.numpy().copy(), np.full(batch, shared)
    dev_pool, dev_tables = pool.to(cuda_device), tables.to(cuda_device)
    dev_lengths = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    dev_new = torch.zeros(batch, dtype=torch.int32, device=cuda_device)
    dev_free = free.to(cuda_device)
    fused = torch.zeros((most, heads * group + 2 * heads, dim), dtype=torch.bfloat16, device=cuda_device)
    query, key, value = fused.split([heads * group, heads, heads], dim=1)
    step = extend_block_tables(dev_tables, dev_lengths, dev_new, dev_free, page_size=page, max_tokens=most)
    out = torch.full((most, heads * group, dim), MARK, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.full((most, heads * group), MARK, device=cuda_device)
    plan = SharedPrefixAttention(query, dev_pool[:, 0], dev_pool[:, 1], dev_tables, step.lengths, page_size=page,
                                 shared_tokens=shared, source_row=batch, query_starts=step.query_starts, out=out, lse=lse)

    def one_step():
        extend_block_tables(dev_tables, dev_lengths, dev_new, dev_free, page_size=page, max_tokens=most, out=step)
        append_rows([key, value], step.slot_map, [dev_pool[:, 0], dev_pool[:, 1]])
        plan()
        dev_lengths.copy_(step.lengths)

    one_step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one_step()
    host_pool = [pool[:, i].float().numpy() for i in range(2)]
    used = 0
    for new in ([30, 1, 20], [1, 1, 1], [0, 5, 33]):
        rows = torch.randn((most, heads * group + 2 * heads, dim), generator=gen).bfloat16()
        fused.copy_(rows)
        dev_new.copy_(torch.tensor(new))
        dev_free[:free.numel() - used].copy_(free[used:])
        out.fill_(MARK)
        lse.fill_(MARK)
        graph.replay()
        host_tables, starts, slot_map, _, lengths, taken = obt.extend(
            host_tables, lengths, new, free.numpy()[used:], page, most)
        used += int(taken[0])
        split = rows.float().split([heads * group, heads, heads], dim=1)
        host_pool = [obt.append(r.numpy(), slot_map, p) for r, p in zip(split[1:], host_pool)]
        want = opa.attend(split[0].double().numpy(), *(p.astype(np.float64) for p in host_pool), host_tables, lengths,
                          page_size=page, shared_tokens=shared, source_row=batch, query_starts=starts)
        np.testing.assert_array_equal(dev_tables.cpu().numpy(), host_tables)
        np.testing.assert_array_equal(dev_lengths.cpu().numpy(), lengths)
        for i, plane in enumerate(host_pool):
            np.testing.assert_array_equal(dev_pool[:, i].float().cpu().numpy(), plane)
        compare((out, lse), want, torch.bfloat16, float(np.abs(host_pool[1]).max()), dim)
    assert donor.min() >= 0 and used < free.numel()
