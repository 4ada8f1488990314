"""Block-table extension and row append on the device against the CPU restatement (exact)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block_tables as obt

pytestmark = pytest.mark.gpu


def _extend_case(seed, requests, page, width, held_high, new_high, free, row_count=None):
    rng = np.random.default_rng(seed)
    row_count = row_count or requests
    tables = rng.integers(-1, 1 << 20, (row_count, width)).astype(np.int32)
    lengths = rng.integers(0, held_high + 1, requests)
    new = rng.integers(0, new_high + 1, requests)
    free_pages = rng.permutation(1 << 20)[:free].astype(np.int32)
    rows = rng.permutation(row_count)[:requests]
    return tables, lengths, new, free_pages, rows


def _check(device, tables, lengths, new, free_pages, rows, page, max_tokens, index=torch.int32, stride=0, **kwargs):
    from ekv_b200.block_tables import extend_block_tables

    want = obt.extend(tables, lengths, new, free_pages, page, max_tokens, rows)
    wide = torch.full((tables.shape[0], tables.shape[1] + stride), -9, dtype=torch.int32, device=device)
    dev_tables = wide[:, :tables.shape[1]]
    dev_tables.copy_(torch.from_numpy(tables))
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(index).to(device)  # noqa: E731
    got = extend_block_tables(dev_tables, to(lengths), to(new), torch.from_numpy(free_pages).to(device),
                              page_size=page, max_tokens=max_tokens, rows=None if rows is None else to(rows), **kwargs)
    np.testing.assert_array_equal(dev_tables.cpu().numpy(), want[0])
    for name, expected in zip(got._fields, want[1:]):
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), expected, err_msg=name)
    assert bool((wide[:, tables.shape[1]:] == -9).all())
    return got


@pytest.mark.parametrize("page", [1, 7, 16, 128])
@pytest.mark.parametrize("requests", [1, 5, 512, 513, 1300])
def test_random_batches(page, requests, cuda_device):
    """Ragged lengths and new tokens, permuted rows, both index types, strided table rows."""
    case = _extend_case(requests + page, requests, page, 40, 30 * page, 4, 5000 // page + requests, requests + 3)
    total = int(case[2].sum())
    index = torch.int64 if requests % 2 else torch.int32
    _check(cuda_device, *case, page, total + 11, index=index, stride=5)


@pytest.mark.parametrize("page", [1, 16])
def test_prompts_spread_over_many_blocks(page, cuda_device):
    """200,000 tokens: every block of the launch places its slice, requests span slices."""
    tables, lengths, new, free, rows = _extend_case(3, 37, page, 24000 // page, 9000, 12000, 300000 // page)
    _check(cuda_device, tables, lengths, new, free, rows, page, int(new.sum()) + 4097)


@pytest.mark.parametrize("short", ["pages", "tokens"])
def test_grants_stop_at_the_first_request_that_does_not_fit(short, cuda_device):
    tables, lengths, new, free, rows = _extend_case(11, 700, 4, 64, 100, 40, 4000)
    if short == "pages":
        got = _check(cuda_device, tables, lengths, new, free[:1500], rows, 4, int(new.sum()))
        assert 0 < int(got.pages_used) <= 1500
    else:
        got = _check(cuda_device, tables, lengths, new, free, rows, 4, int(new.sum()) // 3)
        assert 0 < int(got.query_starts[-1]) <= int(new.sum()) // 3
    assert int(got.lengths.sum()) < int(lengths.sum() + new.sum())


def test_requests_that_are_passed_over(cuda_device):
    """No new tokens, a negative count, rows outside the table, a full row, a negative length."""
    tables = np.arange(6 * 4, dtype=np.int32).reshape(6, 4)
    lengths = np.array([5, 16, 9, 2, 14, -3, 0, 16])
    new = np.array([0, 1, -4, 3, 3, 2, 16, 0])
    rows = np.array([0, 1, 2, 99, 3, 4, 5, -1])
    _check(cuda_device, tables, lengths, new, np.arange(100, 120, dtype=np.int32), rows, 4, 64, index=torch.int64)


def test_holes_give_no_slot(cuda_device):
    """A negative page, in the table or among the free ones, and a slot past 31 bits."""
    tables = np.full((3, 4), 7, dtype=np.int32)
    tables[0, 0] = -1
    free = np.array([-5, (1 << 31) - 2, 3, 4], dtype=np.int32)
    _check(cuda_device, tables, np.array([2, 0, 3]), np.array([7, 4, 2]), free, None, 4, 20)


def test_empty_batches(cuda_device):
    none = np.zeros(0, dtype=np.int64)
    _check(cuda_device, np.zeros((0, 4), dtype=np.int32), none, none, np.zeros(0, dtype=np.int32), None, 4, 9)
    _check(cuda_device, np.zeros((2, 4), dtype=np.int32), np.array([1, 2]), np.array([1, 1]),
           np.zeros(0, dtype=np.int32), None, 4, 0)


def test_captured_step_follows_its_inputs(cuda_device):
    """A captured extension replayed with other lengths; outputs reused in place of new ones."""
    from ekv_b200.block_tables import extend_block_tables

    tables, lengths, new, free, rows = _extend_case(5, 9, 8, 30, 100, 20, 200)
    dev = [torch.from_numpy(a).to(cuda_device) for a in (tables, lengths, new, free, rows)]
    out = extend_block_tables(*dev[:4], page_size=8, max_tokens=300, rows=dev[4])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        extend_block_tables(*dev[:4], page_size=8, max_tokens=300, rows=dev[4], out=out)
    for seed in (6, 7):
        tables, lengths, new, free, rows = _extend_case(seed, 9, 8, 30, 100, 20, 200)
        for tensor, array in zip(dev, (tables, lengths, new, free, rows)):
            tensor.copy_(torch.from_numpy(array))
        graph.replay()
        want = obt.extend(tables, lengths, new, free, 8, 300, rows)
        np.testing.assert_array_equal(dev[0].cpu().numpy(), want[0])
        for tensor, expected in zip(out, want[1:]):
            np.testing.assert_array_equal(tensor.cpu().numpy(), expected)


@pytest.mark.parametrize("shape,dtype", [((8, 128), torch.bfloat16), ((1, 128), torch.float16), ((3, 40), torch.float32),
                                         ((5,), torch.bfloat16), ((7, 3), torch.uint8), ((2, 6), torch.bfloat16)])
@pytest.mark.parametrize("tokens", [1, 63, 700])
def test_append_matches_the_restatement(shape, dtype, tokens, cuda_device):
    """Rows on and off the 16-byte grid, views of a fused projection, skipped and outside slots."""
    from ekv_b200.block_tables import append_rows

    gen = torch.Generator().manual_seed(tokens)
    slots = 900
    fused = torch.randint(0, 256, (tokens, 3, *shape), generator=gen).to(dtype).to(cuda_device)
    rows = [fused[:, 1], fused[:, 2]]
    pool = torch.randint(0, 256, (slots, 2, *shape), generator=gen).to(dtype).to(cuda_device)
    planes = [pool[:, 0], pool[:, 1]]
    slot_map = torch.randperm(slots, generator=gen)[:tokens]
    slot_map[::5] = -1
    if tokens > 10:
        slot_map[3], slot_map[7] = slots, slots + 5
    want = [obt.append(r.float().cpu().numpy(), slot_map.numpy(), p.float().cpu().numpy())
            for r, p in zip(rows, planes)]
    append_rows(rows, slot_map.to(torch.int32 if tokens % 2 else torch.int64).to(cuda_device), planes)
    for plane, expected in zip(planes, want):
        np.testing.assert_array_equal(plane.float().cpu().numpy(), expected)


def test_append_many_planes_and_nothing(cuda_device):
    from ekv_b200.block_tables import append_rows

    gen = torch.Generator().manual_seed(1)
    rows = [torch.randint(0, 999, (17, 4, 8), generator=gen, dtype=torch.int32).to(cuda_device) for _ in range(256)]
    planes = [torch.zeros((40, 4, 8), dtype=torch.int32, device=cuda_device) for _ in range(256)]
    slot_map = torch.randperm(40, generator=gen)[:17].to(cuda_device)
    append_rows(rows, slot_map, planes)
    for row, plane in zip(rows, planes):
        assert torch.equal(plane[slot_map], row) and int((plane != 0).any(2).any(1).sum()) <= 17
    before = planes[0].clone()
    append_rows([rows[0][:0]], slot_map[:0], planes[:1])
    append_rows([], slot_map, [])
    append_rows([rows[0]], torch.full((17,), -1, device=cuda_device), planes[:1])
    assert torch.equal(planes[0], before)


def test_append_past_32_bit_offsets(cuda_device):
    """A plane of more than 2^32 bytes: the highest slots are reached."""
    from ekv_b200.block_tables import append_rows

    slots = (1 << 32) // 2048 + 100
    plane = torch.empty((slots, 8, 128), dtype=torch.bfloat16, device=cuda_device)
    plane[-1].zero_()
    rows = torch.randn(3, 8, 128, device=cuda_device).bfloat16()
    append_rows([rows], torch.tensor([slots - 1, slots - 3, 0], device=cuda_device), [plane])
    assert torch.equal(plane[[slots - 1, slots - 3, 0]], rows)


def test_refusals_on_the_device(cuda_device):
    from ekv_b200.block_tables import append_rows, extend_block_tables

    tables = torch.zeros((2, 4), dtype=torch.int32, device=cuda_device)
    two = torch.ones(2, dtype=torch.int32, device=cuda_device)
    free = torch.arange(8, dtype=torch.int32, device=cuda_device)
    out = extend_block_tables(tables, two, two, free, page_size=4, max_tokens=8)
    with pytest.raises(ValueError, match="overlaps an input"):
        extend_block_tables(tables, out.lengths, two, free, page_size=4, max_tokens=8, out=out)
    with pytest.raises(ValueError, match="CUDA tensor"):
        extend_block_tables(tables, two.cpu(), two, free, page_size=4, max_tokens=8)
    plane = torch.zeros((4, 2, 8), device=cuda_device)
    with pytest.raises(TypeError, match="dtype"):
        append_rows([torch.zeros((2, 2, 8), device=cuda_device).half()], two, [plane])
    with pytest.raises(ValueError, match="overlap"):
        append_rows([torch.zeros((2, 2, 8), device=cuda_device)], two, [plane[:1].expand(4, 2, 8)])


@pytest.mark.parametrize("short", ["pages", "tokens"])
@pytest.mark.parametrize("requests,closing", [(2049, 500), (2049, 1024), (2049, 2048), (3100, 1023), (3100, 1500),
                                              (5000, 3), (5000, 2500), (5000, 4999)])
def test_nothing_is_granted_behind_a_large_request(short, requests, closing, cuda_device):
    """One request needs more than is left and the small ones behind it would not: they get nothing either,
    however many passes of 1024 requests lie between."""
    page = 4
    tables, lengths, new, free, rows = _extend_case(requests + closing, requests, page, 64, 100, 3, 4 * requests)
    new[closing] = 120
    need = lambda n: int((-(-(lengths + new) // page) + -lengths // page)[:n].sum())  # noqa: E731
    if short == "pages":
        free, most = free[:need(closing) + 20], int(new.sum())
    else:
        most = int(new[:closing].sum()) + 100
    got = _check(cuda_device, tables, lengths, new, free, rows, page, most)
    assert int(got.query_starts[-1]) == int(new[:closing].sum()) and int(got.pages_used) == need(closing)
    np.testing.assert_array_equal(got.lengths.cpu().numpy()[closing:], lengths[closing:])
