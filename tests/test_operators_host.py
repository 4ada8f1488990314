"""Argument checks of the block-table, append and shared-prefix attention calls, without a GPU."""

from __future__ import annotations

import ctypes as ct

import numpy as np
import pytest
import torch

from oracle import block_tables as obt
from oracle import prefix_attention as opa


@pytest.fixture
def host(monkeypatch):
    """The modules with the device check passing for CPU tensors and launches refused."""
    from ekv_b200 import block_tables, prefix_attention

    def no_launch(name, *args):
        raise AssertionError(f"{name} was launched")

    for module in (block_tables, prefix_attention):
        monkeypatch.setattr(module, "require_cuda", lambda tensors, device=None: torch.device("cuda", 0))
        monkeypatch.setattr(module, "call", no_launch)
        monkeypatch.setattr(module, "stream_handle", lambda device: 0)
    monkeypatch.setattr(prefix_attention, "torch_binding", lambda: None, raising=False)
    monkeypatch.setattr(block_tables, "torch_binding", lambda: None, raising=False)
    return block_tables, prefix_attention


def _tables():
    return dict(block_tables=torch.zeros((3, 4), dtype=torch.int32), lengths=torch.ones(3, dtype=torch.int32),
                new_tokens=torch.ones(3, dtype=torch.int32), free_pages=torch.arange(5, dtype=torch.int32),
                page_size=4, max_tokens=8)


@pytest.mark.parametrize("change,error,match", [
    (dict(page_size=0), ValueError, "page_size"),
    (dict(page_size=True), ValueError, "page_size"),
    (dict(page_size=1 << 30), ValueError, "2\\^31"),
    (dict(max_tokens=-1), ValueError, "max_tokens"),
    (dict(block_tables=torch.zeros((3, 4), dtype=torch.int64)), TypeError, "int32"),
    (dict(free_pages=torch.zeros(5, dtype=torch.int64)), TypeError, "int32"),
    (dict(block_tables=torch.zeros((4, 3), dtype=torch.int32).t()), ValueError, "contiguous rows"),
    (dict(block_tables=torch.zeros((1, 4), dtype=torch.int32).expand(3, 4)), ValueError, "overlap"),
    (dict(new_tokens=torch.ones(2, dtype=torch.int32)), ValueError, "3 entries"),
    (dict(lengths=torch.ones(3)), TypeError, "int32 or int64"),
    (dict(lengths=torch.ones((3, 1), dtype=torch.int32)), ValueError, "one-dimensional"),
    (dict(lengths=torch.ones(6, dtype=torch.int32)[::2]), ValueError, "contiguous"),
    (dict(rows=torch.zeros(4, dtype=torch.int64)), ValueError, "3 entries"),
])
def test_extend_refuses(change, error, match, host):
    with pytest.raises(error, match=match):
        host[0].extend_block_tables(**{**_tables(), **change})


def test_extend_refuses_outputs_that_do_not_match(host):
    args = _tables()
    flat = torch.zeros(64, dtype=torch.int32)
    good = host[0].TableExtension(flat[:4], flat[8:16], flat[16:24], flat[24:27], flat[28:29])
    for name, tensor in (("slot_map", flat[8:15]), ("pages_used", flat[28:30]), ("lengths", args["lengths"])):
        with pytest.raises(ValueError):
            host[0].extend_block_tables(**args, out=good._replace(**{name: tensor}))
    with pytest.raises(TypeError):
        host[0].extend_block_tables(**args, out=good._replace(positions=torch.zeros(8, dtype=torch.int64)))
    wide = torch.zeros((3, 32), dtype=torch.int32)
    with pytest.raises(ValueError, match="positions overlaps an input"):  # in the table's last row
        host[0].extend_block_tables(**{**args, "block_tables": wide[:, 4:8]},
                                    out=good._replace(positions=wide[2, :8]))


@pytest.mark.parametrize("change", [
    lambda flat: dict(positions=flat[8:16]),    # the slot map's
    lambda flat: dict(positions=flat[15:23]),   # its last entry
    lambda flat: dict(pages_used=flat[3:4]),    # the starts' last entry
])
def test_extend_refuses_outputs_that_overlap_one_another(change, host):
    flat = torch.zeros(64, dtype=torch.int32)
    good = host[0].TableExtension(flat[:4], flat[8:16], flat[16:24], flat[24:27], flat[27:28])
    with pytest.raises(ValueError, match="tensors of out overlap"):
        host[0].extend_block_tables(**_tables(), out=good._replace(**change(flat)))


@pytest.mark.parametrize("rows,slot_map,planes,error,match", [
    ([torch.zeros(3, 2, 8)], torch.zeros(3, dtype=torch.int32), [], ValueError, "length"),
    ([torch.zeros(3, 2, 8)] * 257, torch.zeros(3, dtype=torch.int32), [torch.zeros(5, 2, 8)] * 257, ValueError, "MAX_PLANES"),
    ([torch.zeros(3, 2, 8)], torch.zeros(4, dtype=torch.int32), [torch.zeros(5, 2, 8)], ValueError, "row shape"),
    ([torch.zeros(3, 2, 8)], torch.zeros(3, dtype=torch.int32), [torch.zeros(5, 2, 4)], ValueError, "row shape"),
    ([torch.zeros(3, 2, 8)], torch.zeros(3), [torch.zeros(5, 2, 8)], TypeError, "int32 or int64"),
    ([torch.zeros(3, 2, 8).half()], torch.zeros(3, dtype=torch.int32), [torch.zeros(5, 2, 8)], TypeError, "dtype"),
    ([torch.zeros(3, 8, 2).transpose(1, 2)], torch.zeros(3, dtype=torch.int32), [torch.zeros(5, 2, 8)], ValueError, "contiguous rows"),
    ([torch.zeros(3, 2, 8), torch.zeros(3, 4, 8)[:, :2]], torch.zeros(3, dtype=torch.int32),
     [torch.zeros(5, 2, 8)] * 2, ValueError, "share one row stride"),
    ([torch.zeros(3, 2, 8)], torch.zeros(3, dtype=torch.int32), [torch.zeros(1, 2, 8).expand(5, 2, 8)], ValueError, "overlap"),
])
def test_append_refuses(rows, slot_map, planes, error, match, host):
    with pytest.raises(error, match=match):
        host[0].append_rows(rows, slot_map, planes)


def _attend():
    return dict(query=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k_plane=torch.zeros(32, 2, 64, dtype=torch.bfloat16),
                v_plane=torch.zeros(32, 2, 64, dtype=torch.bfloat16), block_tables=torch.zeros((3, 4), dtype=torch.int32),
                lengths=torch.ones(3, dtype=torch.int32), page_size=4, shared_tokens=8)


@pytest.mark.parametrize("change,error,match", [
    (dict(query=torch.zeros(3, 4, 64)), TypeError, "bfloat16 or float16"),
    (dict(query=torch.zeros(3, 4, 64).half()), TypeError, "share one dtype"),
    (dict(query=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), ValueError, "64 or 128"),
    (dict(query=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), ValueError, "multiple"),
    (dict(query=torch.zeros(3, 256, dtype=torch.bfloat16)), ValueError, "expected query"),
    (dict(query=torch.zeros(3, 4, 128, dtype=torch.bfloat16)[..., ::2]), ValueError, "last dimension"),
    (dict(query=torch.zeros(3, 4, 65, dtype=torch.bfloat16)[..., :64]), ValueError, "16-byte"),
    (dict(query=torch.zeros(769, dtype=torch.bfloat16)[1:].view(3, 4, 64)), ValueError, "16-byte"),
    (dict(v_plane=torch.zeros(31, 2, 64, dtype=torch.bfloat16)), ValueError, "expected query"),
    (dict(k_plane=torch.zeros(1, 2, 64, dtype=torch.bfloat16).expand(32, 2, 64)), ValueError, "overlap"),
    (dict(out=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), ValueError, "out must have"),
    (dict(out=torch.zeros(3, 4, 64)), TypeError, "share one dtype"),
    (dict(out=torch.zeros(6 * 64, dtype=torch.bfloat16).as_strided((3, 4, 64), (64, 64, 1))), ValueError, "out rows overlap"),
    (dict(lse=torch.zeros(4, 3)), ValueError, "lse"),
    (dict(lse=torch.zeros(1, 4).expand(3, 4)), ValueError, "lse rows overlap"),
    (dict(lse=torch.zeros(6).as_strided((3, 4), (1, 1))), ValueError, "lse rows overlap"),
    (dict(lse=torch.zeros(3, 4).double()), TypeError, "float32"),
    (dict(page_size=0), ValueError, "page_size"),
    (dict(page_size=1 << 29), ValueError, "2\\^31"),
    (dict(block_tables=torch.zeros((3, 1), dtype=torch.int32), page_size=(1 << 31) - 255), ValueError, "2\\^31 - 256"),
    (dict(shared_tokens=17), ValueError, "shared_tokens"),
    (dict(shared_tokens=-1), ValueError, "shared_tokens"),
    (dict(source_row=3), ValueError, "source row"),
    (dict(rows=torch.zeros(2, dtype=torch.int32)), ValueError, "3 entries"),
    (dict(query_starts=torch.zeros(3, dtype=torch.int32)), ValueError, "4 entries"),
    (dict(lengths=torch.ones(2, dtype=torch.int32)), ValueError, "one query token"),
    (dict(query=torch.zeros(1 << 18, 4, 1, dtype=torch.bfloat16).expand(-1, -1, 64)), ValueError, "last dimension"),
    (dict(lengths=torch.ones(1537, dtype=torch.int32), query=torch.zeros(1537, 4, 64, dtype=torch.bfloat16)), ValueError,
     "one call takes"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(scale=float("inf")), ValueError, "scale"),
])
def test_attention_refuses(change, error, match, host):
    with pytest.raises(error, match=match):
        host[1].shared_prefix_attention(**{**_attend(), **change})
    with pytest.raises(error, match=match):
        host[1].SharedPrefixAttention(**{**_attend(), **change})


def test_host_tensors_are_refused(library_path):
    from ekv_b200.block_tables import append_rows, extend_block_tables
    from ekv_b200.prefix_attention import shared_prefix_attention

    with pytest.raises(ValueError, match="CUDA tensor"):
        extend_block_tables(**_tables())
    with pytest.raises(ValueError, match="CUDA tensor"):
        append_rows([torch.zeros(3, 2, 8)], torch.zeros(3, dtype=torch.int32), [torch.zeros(5, 2, 8)])
    with pytest.raises(ValueError, match="CUDA tensor"):
        shared_prefix_attention(**_attend())


def _attention_args(**change):
    """Arguments of ekv_shared_prefix_attention that pass every check but the changed ones."""
    a = dict(query=4096, qs=(512, 64), k=4096, ks=(128, 64), v=4096, vs=(128, 64), slots=32, dtype=0, dim=64,
             query_heads=4, kv_heads=2, tokens=3, batch=3, tables=4096, table_es=4, table_rows=3, width=4, stride=4,
             page=4, lengths=4096, starts=None, shared=8, source=0, scale=1.0, out=4096, os=(512, 64), workspace=None,
             workspace_bytes=0)
    a.update(change)
    return (a["query"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["slots"], a["dtype"], a["dim"],
            a["query_heads"], a["kv_heads"], a["tokens"], a["batch"], a["tables"], a["table_es"], a["table_rows"],
            a["width"], a["stride"], a["page"], None, 8, a["lengths"], 4, a["starts"], 4, a["shared"], a["source"],
            a["scale"], a["out"], *a["os"], None, 0, 0, a["workspace"], a["workspace_bytes"], 0, None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=7), b"dtype"), (dict(dim=96), b"head_dim"), (dict(query_heads=5), b"multiple"),
    (dict(tokens=-1), b"negative"), (dict(page=0), b"page_size"), (dict(shared=17), b"shared_tokens"),
    (dict(source=3), b"source row"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(batch=2), b"one query token"), (dict(query=None), b"null pointer"), (dict(query=4098), b"16-byte"),
    (dict(ks=(127, 64)), b"16-byte"), (dict(table_es=2), b"element size"),
    (dict(tokens=1537, batch=1537), b"ROW_TILES"), (dict(tokens=1 << 20, starts=4096), b"ROW_TILES"),
    (dict(width=1 << 30, page=1, tokens=1500, batch=1500), b"too wide"),
])
def test_c_entry_refuses_before_touching_a_device(change, message, library_path):
    from ekv_b200 import _lib

    lib = _lib.library(str(library_path))
    assert lib.ekv_shared_prefix_attention(*_attention_args(**change)) == -1
    assert message in lib.ekv_error(), lib.ekv_error()
    assert lib.ekv_bitmap_and(None, 1, 0, None, 0, None) == 0 and lib.ekv_error() == b""  # the next call clears it


def test_other_c_entries_refuse_and_pass_empty_work(library_path):
    from ekv_b200 import _lib

    lib = _lib.library(str(library_path))
    p = ct.c_void_p(4096)
    assert lib.ekv_shared_prefix_attention(*_attention_args(tokens=0, batch=0)) == 0
    extend = lambda **c: lib.ekv_extend_block_tables(  # noqa: E731
        p, c.get("rows", 3), c.get("width", 4), 4, None, 8, c.get("lengths", p), 4, p, c.get("new_es", 4), 3, p, 5,
        c.get("page", 4), c.get("tokens", 8), p, p, p, p, c.get("used", p), 0, None)
    for change, message in ((dict(page=0), b"page_size"), (dict(width=1 << 30), b"2^31"), (dict(rows=-1), b"negative"),
                            (dict(tokens=1 << 31), b"2^31"), (dict(lengths=None), b"null"), (dict(new_es=3), b"element"),
                            (dict(used=None), b"null")):
        assert extend(**change) == -1 and message in lib.ekv_error(), (change, lib.ekv_error())
    planes = _lib.u64_array([4096])
    assert lib.ekv_append_rows(planes, planes, 257, 16, 16, 16, p, 4, 1, 1, 0, None) == -1 and b"plane" in lib.ekv_error()
    assert lib.ekv_append_rows(planes, planes, 1, 16, 16, 16, None, 4, 1, 1, 0, None) == -1 and b"null" in lib.ekv_error()
    assert lib.ekv_append_rows(planes, planes, 1, 16, 16, 16, p, 2, 1, 1, 0, None) == -1 and b"element" in lib.ekv_error()
    assert lib.ekv_append_rows(planes, planes, 1, -1, 16, 16, p, 4, 1, 1, 0, None) == -1
    assert lib.ekv_append_rows(planes, planes, 1, 16, 16, 16, None, 4, 0, 1, 0, None) == 0


def test_restatement_known_answers():
    """The CPU restatements at sizes that are checked by hand."""
    tables, starts, slot_map, positions, lengths, used = obt.extend(
        np.array([[5, 0], [6, 0]]), [3, 4], [2, 1], np.array([9, 8]), 4, 5)
    assert tables.tolist() == [[5, 9], [6, 8]] and starts.tolist() == [0, 2, 3] and lengths.tolist() == [5, 5]
    assert slot_map.tolist() == [23, 36, 32, -1, -1] and positions.tolist() == [3, 4, 4, -1, -1] and used.tolist() == [2]
    query = np.zeros((1, 1, 2))
    keys = np.ones((4, 1, 2))
    values = np.arange(8.0).reshape(4, 1, 2)
    out, lse, *_ = opa.attend(query, keys, values, np.array([[1, 0]]), [3], page_size=2, scale=1.0)
    np.testing.assert_allclose(out[0, 0], (values[2, 0] + values[3, 0] + values[0, 0]) / 3)
    np.testing.assert_allclose(lse, np.log(3.0))


@pytest.mark.parametrize("scale", [2.4e38, 2.99e38, 1e-46, -1.0, -0.0])
def test_attention_refuses_scales_that_32_bits_do_not_hold(scale, host, library_path):
    """scale * log2(e), the factor of the kernels, has to be a positive number of 32 bits."""
    from ekv_b200 import _lib

    with pytest.raises(ValueError, match="scale"):
        host[1].shared_prefix_attention(**_attend(), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        host[1].SharedPrefixAttention(**_attend(), scale=scale)
    lib = _lib.library(str(library_path))
    assert lib.ekv_shared_prefix_attention(*_attention_args(scale=scale, tokens=0, batch=0)) == -1
    assert b"scale" in lib.ekv_error()


@pytest.mark.parametrize("scale", [2.3e38, 1.5e-45])
def test_the_ends_of_the_scales_are_taken(scale, host, library_path):
    from ekv_b200 import _lib

    with pytest.raises(AssertionError, match="was launched"):
        host[1].shared_prefix_attention(**_attend(), scale=scale)
    assert _lib.library(str(library_path)).ekv_shared_prefix_attention(*_attention_args(scale=scale, tokens=0, batch=0)) == 0
    assert np.isfinite(np.float32(scale) * np.float32(1.4426950408889634)) and np.float32(scale) > 0


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _sharing():
    """Calls whose outputs share memory with an input or one another, and what the refusal says."""
    tokens, wide = _bf16(4, 4, 64), _bf16(3, 8, 64)
    flat, plane, words = _bf16(1024), _bf16(32, 2, 64), torch.zeros(64, dtype=torch.int32)
    yield dict(query=tokens[:3], out=tokens[1:]), "out overlaps query"
    yield dict(query=flat[:768].view(3, 4, 64), out=flat[8:776].view(3, 4, 64)), "out overlaps query"
    yield dict(query=wide[:, :4], out=wide[:, 2:6]), "out overlaps query"
    yield dict(query=wide[:, :4], out=wide.view(-1)[:768].view(3, 4, 64)), "out overlaps query"  # other strides
    yield dict(query=tokens[:1].expand(3, -1, -1), out=tokens[:3]), "out overlaps query"
    yield dict(k_plane=plane, out=plane.view(-1)[-768:].view(3, 4, 64)), "out overlaps a plane"
    yield dict(v_plane=plane, out=plane.view(-1)[:768].view(3, 4, 64)), "out overlaps a plane"
    yield dict(v_plane=plane, lse=plane.view(-1)[:24].view(torch.float32).view(3, 4)), "lse overlaps a plane"
    yield dict(query=tokens[:3], lse=tokens.view(-1)[744:768].view(torch.float32).view(3, 4)), "lse overlaps query"
    yield dict(out=tokens[:3], lse=tokens.view(-1)[744:768].view(torch.float32).view(3, 4)), "out and lse overlap"
    yield dict(lengths=words[10:13], lse=words[2:14].view(torch.float32).view(3, 4)), "lse overlaps an index"
    yield dict(block_tables=words[:12].view(3, 4), lse=words[11:23].view(torch.float32).view(3, 4)), "lse overlaps an index"
    yield dict(rows=words[:3], lse=words[:12].view(torch.float32).view(3, 4)), "lse overlaps an index"
    yield dict(query_starts=words[8:12], lse=words[:12].view(torch.float32).view(3, 4)), "lse overlaps an index"


@pytest.mark.parametrize("change,match", list(_sharing()))
def test_attention_refuses_outputs_in_memory_that_is_read(change, match, host):
    with pytest.raises(ValueError, match=match):
        host[1].shared_prefix_attention(**{**_attend(), **change})
    with pytest.raises(ValueError, match=match):
        host[1].SharedPrefixAttention(**{**_attend(), **change})


def _beside():
    tokens, wide, flat = _bf16(3, 4, 64), _bf16(3, 12, 64), torch.zeros(1024)
    pool, words = _bf16(32, 3, 2, 64), torch.zeros(64, dtype=torch.int32)
    yield dict(query=tokens, out=tokens)
    yield dict(query=wide[:, :4], out=wide[:, :4])
    yield dict(query=wide[:, :4], out=wide[:, 4:8])  # interleaved
    yield dict(query=wide[:, 8:], out=wide[:, :4])
    yield dict(query=wide[:, :2], out=wide[:, 3:5], k_plane=_bf16(32, 1, 64), v_plane=_bf16(32, 1, 64))
    yield dict(k_plane=pool[:, 0], v_plane=pool[:, 1], query=_bf16(3, 2, 64), out=pool[:3, 2])  # a third plane of the pool
    yield dict(out=flat[:384].view(torch.bfloat16).view(3, 4, 64), lse=flat[384:396].view(3, 4))
    yield dict(lse=words[:12].view(torch.float32).view(4, 3).t(), lengths=words[12:15], rows=words[15:18])


@pytest.mark.parametrize("change", list(_beside()))
def test_attention_takes_outputs_beside_what_is_read(change, host):
    with pytest.raises(AssertionError, match="was launched"):
        host[1].shared_prefix_attention(**{**_attend(), **change})


def test_shared_elements_are_found():
    """Random views of one buffer against the set of their elements; the compiled form agrees."""
    from ekv_b200 import _lib
    from ekv_b200.prefix_attention import _collide

    compiled = getattr(_lib.torch_binding(), "collide", _collide)
    rng = np.random.default_rng(2)
    buffer = torch.zeros(600, dtype=torch.int16)
    shared = exact = 0
    for _ in range(6000):
        steps = rng.integers(1, 40, 2)
        views = []
        for _ in range(2):
            if rng.random() < 0.2:
                steps = rng.integers(0, 40, 2)
            shape, width = rng.integers(1, 5, 2), int(rng.integers(1, 6))
            views.append(buffer.as_strided((*shape, width), (*steps, 1), int(rng.integers(0, 250))))
        a, b = ({int(e) for e in torch.arange(600).as_strided(v.shape, v.stride(), v.storage_offset()).reshape(-1)} for v in views)
        found = _collide(*views)
        assert found == compiled(*views) and (found or not a & b)
        shared += bool(a & b)
        exact += not found and max(min(a), min(b)) <= min(max(a), max(b))  # interleaved
    assert shared > 500 and exact > 100
