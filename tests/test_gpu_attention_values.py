"""Shared-prefix attention on the device: values that the sums have to hold.

Every comparison here also asks that a result is finite where the definition is (a comparison with NaN
is false, so an error bound alone lets one pass).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import prefix_attention as opa
from test_gpu_prefix_attention import E, MARK, Case, compare

pytestmark = pytest.mark.gpu

# What each takes through the kernels: requests of few rows alone; a prefix in tiles of up to 128 rows and
# of more; new tokens of 17 rows and more, up to several tiles of rows.
SHAPES = {
    "decode": dict(lengths=[900, 65, 2049], shared=0, group=4),
    "decode, 16 rows": dict(lengths=[700, 1300], shared=0, group=16),
    "short prefix, few rows": dict(lengths=[1030, 1025], shared=1024, group=4),
    "prefix, 48 rows": dict(lengths=[1290 + 3 * b for b in range(12)], shared=1280, group=4),
    "prefix, 320 rows": dict(lengths=[1025 + b for b in range(40)], shared=1024, group=8),
    "drafts": dict(lengths=[400, 333, 290], new=[5, 5, 5], shared=256, group=4),
    "prompts": dict(lengths=[700, 500, 900], new=[130, 70, 300], shared=200, group=3),
    "prompts, no prefix": dict(lengths=[300, 20, 129], new=[300, 20, 129], shared=0, group=2),
}


def _np(tensor):
    return tensor.detach().double().cpu().numpy()


def _slots(case, request, count):
    """Slots of the first ``count`` positions of a request."""
    position, slots = np.arange(count), case.k.shape[0]
    own = opa.slots_of(case.tables[request].numpy(), position, case.page, slots)
    donor = opa.slots_of(case.tables[case.source].numpy(), position, case.page, slots)
    return torch.from_numpy(np.where(position < case.shared, donor, own))


def finite_where_defined(got, want):
    out, lse = _np(got[0]), _np(got[1])
    held = ~np.isnan(want[0]).all((1, 2))
    assert np.isfinite(out[held]).all()
    assert (np.isfinite(lse[held]) == np.isfinite(want[1][held])).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_results_are_finite(shape, dim, dtype, cuda_device):
    case = Case(**SHAPES[shape], heads=2, dim=dim, dtype=dtype, tail=3 if "new" in SHAPES[shape] else 0)
    got, want = case.run(cuda_device), case.want()
    finite_where_defined(got, want)
    compare(got, want, dtype, float(case.v.double().abs().max()), dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_items_that_the_halves_of_a_block_share(dim, dtype, cuda_device):
    """Items of 20 and 60 rows, eight tiles of them a block: its halves take the tiles in turn and each joins half of the
    columns of both.  Scores grow along the positions, so that either half has rescaled its sums just before."""
    case = Case(lengths=[9000, 8033, 9900], shared=4000, heads=8, group=20, dim=dim, dtype=dtype, page=64, spread=0.5)
    for request, length in enumerate(case.lengths.tolist()):
        slots = _slots(case, request, length)
        ramp = torch.linspace(0.2, 8.0, length)[:, None, None]
        head = case.query[request].reshape(8, 20, dim)[:, 0].float()
        case.k[slots] = (case.k[slots].float() * 0.2 + head[None] * ramp).to(dtype)
    got, want = case.run(cuda_device), case.want()
    finite_where_defined(got, want)
    compare(got, want, dtype, float(case.v.double().abs().max()), dim)
    for _ in range(5):
        again = case.run(cuda_device)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


def test_between_matrix_products(cuda_device):
    """Calls right behind and before library products on one stream, eagerly and in a graph: tensor memory that either
    holds is free again when the other takes it."""
    from ekv_b200.prefix_attention import SharedPrefixAttention

    case = Case(**SHAPES["prefix, 320 rows"], heads=2, dim=128)
    dev = [t.to(cuda_device) for t in (case.query, case.k, case.v, case.tables, case.lengths)]
    plan = SharedPrefixAttention(*dev, page_size=case.page, shared_tokens=case.shared, source_row=case.source, return_lse=True)
    small, large = (torch.randn(n, n, device=cuda_device).bfloat16() for n in (512, 4096))

    def step():
        products = []
        for matrix in (small, large, small):
            products.append(matrix @ matrix)
            plan()
        return products

    first = step()
    want = plan.out.clone(), plan.lse.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(5):
        again = step()
        assert torch.equal(plan.out, want[0]) and torch.equal(plan.lse, want[1])
        plan.out.zero_()
        graph.replay()
        assert torch.equal(plan.out, want[0]) and torch.equal(plan.lse, want[1])
        for products in (again, captured):
            assert all(torch.equal(a, b) for a, b in zip(products, first))
    compare((plan.out, plan.lse), case.want(), case.dtype, float(case.v.double().abs().max()), 128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_scores_far_beyond_the_exponent(shape, dim, dtype, cuda_device):
    """Scores of 2^30 to 2^32, exact in 32 bits and further apart than any rounding: the mean of V over the
    positions of the largest.  (A maximum rounded to 32 bits and an exact score differ by up to 2^8 here.)"""
    gen = torch.Generator().manual_seed(dim)
    case = Case(**SHAPES[shape], heads=1, dim=dim, dtype=dtype)
    case.query.zero_()
    case.k.zero_()
    case.query[..., :16] = 2.0 ** 15
    values = (1 + torch.randint(1, 100, (case.k.shape[0], 1, 1), generator=gen) / 128) * 2.0 ** 15
    values[torch.rand(values.shape, generator=gen) < 0.3] *= -1
    case.k[..., :16] = values.to(dtype)
    got, want = case.run(cuda_device, scale=0.125), case.want(scale=0.125)
    finite_where_defined(got, want)
    expected, lse, weight, _, seen = want
    # Weights are 1 and 0: what is rounded are the sums and the result, and the maximum of lse.
    tolerance = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    tolerance = tolerance * np.abs(expected) + (2 * seen[:, None, None] + 8) * E * weight + 2.0 ** -25
    assert (np.abs(_np(got[0]) - expected) <= tolerance).all()
    assert (np.abs(_np(got[1]) - lse) <= 8 * E * np.abs(lse)).all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("power,dtype", [*((n, t) for n in (20, 24, 26, 27, 28, 30) for t in (torch.bfloat16, torch.float16)),
                                         (34, torch.bfloat16)])
def test_large_scores_stay_a_mean_of_v(power, shape, dtype, cuda_device):
    """Scores about 2^power that grow by a step of their 32 bits from position to position: which of the last takes
    the weight is rounding's choice, but the result is a mean of V."""
    case = Case(**SHAPES[shape], heads=1, dim=64, dtype=dtype)
    case.query.zero_()
    case.k.zero_()
    base, step = 2.0 ** (power // 2), max(2.0 ** (power - 23), 1.0)
    case.query[..., 0], case.query[..., 1] = base, 1.0
    case.k[..., 0] = 1.25 * 2.0 ** (power - power // 2)
    for b, length in enumerate(case.lengths.tolist()):
        case.k[_slots(case, b, length), :, 1] = (step * (torch.arange(length) % 250)[:, None]).clamp(max=60000).to(dtype)
    got, want = case.run(cuda_device, scale=1.0), case.want(scale=1.0)
    finite_where_defined(got, want)
    largest = float(case.v.double().abs().max())
    out = _np(got[0])
    assert (np.abs(out) <= largest * (1 + 2.0 ** -7)).all(), np.abs(out).max()
    # The maximum is the scores', off by the rounding of a sum of two, of the scale and of the product.
    assert (np.abs(_np(got[1]) - want[1]) <= 8 * E * np.abs(want[1]) + 1e-3).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_flat_tail_keeps_its_weight_in_fp16(shape, dim, cuda_device):
    """The first position of every 128 has V = 0 and takes all but 2^-26 of each other one's weight, whose V is
    large.  fp16 holds weights down to steps of 2^-24; they refer to 2^-7 of the maximum (or less), so each is off by
    2^-32 of the largest, beside half a step of its own."""
    case = Case(**SHAPES[shape], heads=1, dim=dim, dtype=torch.float16)
    case.query.zero_()
    case.query[..., 0] = 4.0
    case.k.zero_()
    case.v[:] = (case.v.float().abs() * 64 + 512).half()
    for b, length in enumerate(case.lengths.tolist()):
        sharp = _slots(case, b, length)[::128]
        case.k[sharp, :, 0] = 4.5  # 18 = 25.97 log 2
        case.v[sharp] = 0.0
    got, want = case.run(cuda_device, scale=1.0), case.want(scale=1.0)
    finite_where_defined(got, want)
    expected, lse, weight, _, seen = want
    v_max, u = float(case.v.double().max()), 2.0 ** -11
    total = np.exp(lse - 18.0)[..., None]  # the sum of the weights, the largest 1
    # Scores are exact (one product); an exponent of 26 is off by 4 e of itself, the sums by n e.
    inner = (2 * seen[:, None, None] + 200) * E
    tolerance = u * (weight + np.abs(expected)) * (1 + 2 * u) + inner * weight
    tolerance = tolerance + seen[:, None, None] * 2.0 ** -32 * v_max / total + 2.0 ** -25
    excess = np.abs(_np(got[0]) - expected) - tolerance
    assert excess.max() <= 0, (excess.max(), float((np.abs(_np(got[0]) - expected) / tolerance).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_whose_scores_are_all_minus_infinity(dtype, cuda_device):
    """By the definition 0 / 0, with a log-sum-exp of minus infinity; a row that sees no position has zeros, and one
    finite score is enough for a result."""
    # Decode: all of it odd; one finite; nothing seen; a table row that holds no page; odd shared positions.
    case = Case(lengths=[40, 41, 0, 37, 90], shared=0, dtype=dtype, heads=1, group=4, dim=64)
    case.query.abs_().clamp_(min=0.5)
    case.tables[3] = -1
    for request, count in ((0, 40), (1, 40)):
        case.k[_slots(case, request, count), :, 3] = -float("inf")
    out, lse = (_np(t) for t in case.run(cuda_device))
    assert np.isnan(out[0]).all() and np.isneginf(lse[0]).all()
    assert np.isfinite(out[[1, 4]]).all() and np.isfinite(lse[[1, 4]]).all()
    np.testing.assert_allclose(out[1], np.broadcast_to(_np(case.v[_slots(case, 1, 41)[40]]), out[1].shape), rtol=2.0 ** -7)
    assert (out[[2, 3]] == 0).all() and np.isneginf(lse[[2, 3]]).all()
    # Prompts: the first 30 tokens of request 0 see odd keys only.
    case = Case(lengths=[200, 150], new=[200, 100], shared=0, dtype=dtype, heads=1, group=4, dim=64)
    case.query.abs_().clamp_(min=0.5)
    case.k[_slots(case, 0, 30), :, 5] = -float("inf")
    out, lse = (_np(t) for t in case.run(cuda_device))
    assert np.isnan(out[:30]).all() and np.isneginf(lse[:30]).all()
    assert np.isfinite(out[30:]).all() and np.isfinite(lse[30:]).all()
    # A prefix of odd keys: the request inside it sees nothing else, those behind it do.
    case = Case(lengths=[300, 301, 350] + [310] * 9, shared=300, dtype=dtype, heads=1, group=4, dim=64)
    case.query.abs_().clamp_(min=0.5)
    case.k[_slots(case, 0, 300), :, 7] = -float("inf")
    out, lse = (_np(t) for t in case.run(cuda_device))
    assert np.isnan(out[0]).all() and np.isneginf(lse[0]).all()
    assert np.isfinite(out[1:]).all() and np.isfinite(lse[1:]).all()


@pytest.mark.parametrize("scale", [2.3e38, 1.5e-45])
@pytest.mark.parametrize("shape", ["decode", "prefix, 48 rows", "prompts"])
def test_the_ends_of_the_scales(shape, scale, cuda_device):
    """Scores of 0 at the largest scale, and any at the smallest, weigh every position alike."""
    case = Case(**SHAPES[shape], heads=1, dim=64)
    if scale > 1:
        case.query.zero_()
    got, want = case.run(cuda_device, scale=scale), case.want(scale=scale)
    finite_where_defined(got, want)
    compare(got, want, case.dtype, float(case.v.double().abs().max()), 64)
    with pytest.raises(ValueError, match="scale"):
        case.run(cuda_device, scale=2.4e38)
    with pytest.raises(ValueError, match="scale"):
        case.run(cuda_device, scale=1e-46)


def test_outputs_in_shared_buffers(cuda_device):
    """Outputs interleaved with the query or the planes are taken, ones in memory that is read are refused."""
    case = Case(lengths=[60, 20, 300], shared=30, heads=2, group=2, dim=64)
    dev = [t.to(cuda_device) for t in (case.k, case.v, case.tables, case.lengths)]
    fused = torch.full((3, 12, 64), MARK, dtype=case.dtype, device=cuda_device)
    fused[:, 4:8] = case.query.to(cuda_device)
    got = case.run(cuda_device)

    def run(**args):
        from ekv_b200.prefix_attention import shared_prefix_attention

        return shared_prefix_attention(fused[:, 4:8], *dev, page_size=16, shared_tokens=30, source_row=case.source, **args)

    assert torch.equal(run(out=fused[:, 8:]), got[0])
    assert bool((fused[:, :4] == MARK).all()) and torch.equal(fused[:, 4:8].cpu(), case.query)
    for out in (fused[:, 3:7], fused.view(-1)[:768].view(3, 4, 64), dev[0].view(-1)[:768].view(3, 4, 64)):
        with pytest.raises(ValueError, match="out overlaps"):
            run(out=out)
    with pytest.raises(ValueError, match="out and lse overlap"):
        run(out=fused[:, :4], lse=fused.view(-1)[:24].view(torch.float32).view(3, 4))
    assert torch.equal(run(out=fused[:, 4:8]), got[0])


@pytest.mark.parametrize("new", [None, [1, 5, 0, 20]])
def test_query_rows_far_behind_the_last_token(new, cuda_device):
    """A step captured for 600 tokens that holds a few: NaN behind the last query, outputs there left alone."""
    from ekv_b200.prefix_attention import SharedPrefixAttention

    case = Case(lengths=[310, 330, 300, 420], shared=300, new=new or [1] * 4, heads=2, group=4, dim=64)
    count = case.query.shape[0]
    query = torch.full((600, *case.query.shape[1:]), float("nan"), dtype=case.dtype, device=cuda_device)
    query[:count] = case.query.to(cuda_device)
    out, lse = torch.full_like(query, MARK), torch.full(query.shape[:2], MARK, device=cuda_device)
    dev = [t.to(cuda_device) for t in (case.k, case.v, case.tables, case.lengths)]
    plan = SharedPrefixAttention(query, *dev, page_size=16, shared_tokens=300, source_row=case.source,
                                 query_starts=case.starts.to(cuda_device), out=out, lse=lse)
    graph = torch.cuda.CUDAGraph()
    plan()
    with torch.cuda.graph(graph):
        plan()
    out.fill_(MARK)
    lse.fill_(MARK)
    graph.replay()
    assert bool((out[count:] == MARK).all()) and bool((lse[count:] == MARK).all())
    got, want = (out[:count], lse[:count]), case.want()
    finite_where_defined(got, want)
    compare(got, want, case.dtype, float(case.v.double().abs().max()), 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,heads,group,dim,new", [
    ([131072], 1, 4, 128, None), ([32768, 40001, 3], 1, 1, 64, None), ([33000, 20000], 2, 4, 128, [3, 1]),
    ([40000, 9000], 1, 4, 64, [30, 2]),
])
def test_long_own_contexts_in_few_heads(lengths, heads, group, dim, new, dtype, cuda_device):
    """One request spread over all warps or blocks, whose parts the join walks one by one; without a prefix."""
    case = Case(lengths=lengths, shared=0, heads=heads, group=group, dim=dim, dtype=dtype, new=new, page=64, spread=3.0)
    got, want = case.run(cuda_device), case.want()
    finite_where_defined(got, want)
    compare(got, want, dtype, float(case.v.double().abs().max()), dim)
    again = case.run(cuda_device)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
