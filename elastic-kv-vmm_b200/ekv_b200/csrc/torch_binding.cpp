// Compiled Python binding of the per-call residency lookups and gathers (optional).
//
// resolve_resident, lookup_slots, the batched shared-prefix resolver,
// gather_rows / gather_rows_planes, append_rows and shared_prefix_attention are
// called once per layer per decode step (extend_block_tables once per step)
// through the Python API.  Through ctypes a call costs ~10 us of
// host time (reading ~30 tensor attributes in Python and marshalling ~28
// arguments); here the tensors arrive as at::Tensor and their pointers,
// strides and the current stream are read in C++.  The kernels are reached
// through the SAME C entry points of libekv_b200.so: Python hands over their
// addresses once (bind), so this module does not link against the library.
//
// Only the well-formed calls are handled here: every tensor on one CUDA
// device, supported dtypes and shapes.  Anything else returns kNotHandled and
// the Python wrapper runs its checked ctypes path, which raises the documented
// errors -- so error types and messages stay exactly those of the Python API.
#include <torch/extension.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <optional>
#include <utility>
#include <vector>

#include "ekv_kernels.h"

namespace {

constexpr int kNotHandled = 1;  // ask the caller to take its checked path
constexpr int kKernelError = -1;

decltype(&ekv_resolve_resident) g_resolve = nullptr;
decltype(&ekv_lookup_slots) g_lookup = nullptr;
decltype(&ekv_resolve_shared_blocks) g_shared = nullptr;
decltype(&ekv_gather_rows) g_gather = nullptr;
decltype(&ekv_gather_rows_planes) g_gather_planes = nullptr;
decltype(&ekv_extend_block_tables) g_extend = nullptr;
decltype(&ekv_append_rows) g_append = nullptr;
decltype(&ekv_shared_prefix_workspace) g_workspace = nullptr;
decltype(&ekv_shared_prefix_attention) g_attention = nullptr;

void bind(int64_t resolve, int64_t lookup, int64_t shared, int64_t gather, int64_t gather_planes, int64_t extend,
          int64_t append, int64_t workspace, int64_t attention) {
    g_resolve = reinterpret_cast<decltype(&ekv_resolve_resident)>(resolve);
    g_lookup = reinterpret_cast<decltype(&ekv_lookup_slots)>(lookup);
    g_shared = reinterpret_cast<decltype(&ekv_resolve_shared_blocks)>(shared);
    g_gather = reinterpret_cast<decltype(&ekv_gather_rows)>(gather);
    g_gather_planes = reinterpret_cast<decltype(&ekv_gather_rows_planes)>(gather_planes);
    g_extend = reinterpret_cast<decltype(&ekv_extend_block_tables)>(extend);
    g_append = reinterpret_cast<decltype(&ekv_append_rows)>(append);
    g_workspace = reinterpret_cast<decltype(&ekv_shared_prefix_workspace)>(workspace);
    g_attention = reinterpret_cast<decltype(&ekv_shared_prefix_attention)>(attention);
}

int index_size(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kInt: return 4;
        case at::kLong: return 8;
        default: return 0;
    }
}

// All defined tensors CUDA on one device; the device index, or -1.
int common_device(std::initializer_list<const at::Tensor*> tensors) {
    int device = -1;
    for (const at::Tensor* t : tensors) {
        if (!t || !t->defined()) continue;
        if (!t->is_cuda()) return -1;
        const int here = t->get_device();
        if (device < 0) {
            device = here;
        } else if (here != device) {
            return -1;
        }
    }
    return device;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

int resolve_resident(const at::Tensor& topk, const at::Tensor& table, const at::Tensor& mapping,
                     const at::Tensor& rows, const at::Tensor& lengths, const at::Tensor& selected,
                     const at::Tensor& output, int64_t block_size) {
    if (!g_resolve || topk.dim() != 3) return kNotHandled;
    const int64_t width = topk.size(2) * block_size;
    if (selected.numel() == 0 || width == 0) return 0;  // no-op, as the reference
    const int device = common_device({&topk, &table, &mapping, &rows, &lengths, &selected, &output});
    if (device < 0 || output.scalar_type() != at::kInt || table.dim() != 2 || output.dim() != 3) return kNotHandled;
    const int es_topk = index_size(topk), es_table = index_size(table), es_map = index_size(mapping);
    const int es_rows = index_size(rows), es_len = index_size(lengths), es_sel = index_size(selected);
    if (!es_topk || !es_table || !es_map || !es_rows || !es_len || !es_sel) return kNotHandled;
    const int rc = g_resolve(
        topk.data_ptr(), es_topk, topk.stride(1), topk.stride(2), topk.size(2),
        table.data_ptr(), es_table, table.stride(0), table.stride(1),
        mapping.data_ptr(), es_map, mapping.stride(0),
        rows.data_ptr(), es_rows, rows.stride(0),
        lengths.data_ptr(), es_len, lengths.stride(0),
        selected.data_ptr(), es_sel, selected.stride(0), selected.numel(),
        output.data_ptr<int32_t>(), output.stride(1), output.stride(2),
        block_size, device, stream_of(device));
    return rc == 0 ? 0 : kKernelError;
}

bool rows_of(const std::optional<at::Tensor>& t, int device, at::ScalarType dtype, int64_t batch) {
    if (!t) return true;
    return t->is_cuda() && t->get_device() == device && t->scalar_type() == dtype && t->dim() >= 1 &&
           t->size(0) == batch && t->stride(-1) == 1;
}

// Returns (status, slots, miss, miss_list, miss_count); outputs not given are allocated.
py::tuple lookup_slots(const at::Tensor& residency_map, const at::Tensor& topk,
                       const std::optional<at::Tensor>& lengths, std::optional<at::Tensor> slots,
                       std::optional<at::Tensor> miss, std::optional<at::Tensor> miss_list,
                       std::optional<at::Tensor> miss_count, bool compact) {
    auto not_handled = [] { return py::make_tuple(kNotHandled, py::none(), py::none(), py::none(), py::none()); };
    if (!g_lookup || residency_map.dim() != 2 || topk.dim() != 2 || residency_map.size(0) != topk.size(0)) {
        return not_handled();
    }
    const at::Tensor* len_ptr = lengths ? &*lengths : nullptr;
    const int device = common_device({&residency_map, &topk, len_ptr});
    if (device < 0 || residency_map.stride(1) != 1 || topk.stride(1) != 1) return not_handled();
    const int es_map = index_size(residency_map), es_topk = index_size(topk);
    const int es_len = lengths ? index_size(*lengths) : 4;
    if (!es_map || !es_topk || !es_len) return not_handled();
    const int64_t batch = topk.size(0), k = topk.size(1);
    if (lengths && (lengths->dim() != 1 || lengths->size(0) != batch || lengths->stride(0) != 1)) {
        return not_handled();
    }
    const auto options = residency_map.options();
    if (!slots) slots = at::empty({batch, k}, options.dtype(at::kInt));
    if (!miss) miss = at::empty({batch, k}, options.dtype(at::kBool));
    if (compact) {
        if (!miss_list) miss_list = at::empty({batch, k}, options.dtype(at::kInt));
        if (!miss_count) miss_count = at::empty({batch}, options.dtype(at::kInt));
    }
    if (!rows_of(slots, device, at::kInt, batch) || !rows_of(miss, device, at::kBool, batch) ||
        !rows_of(miss_list, device, at::kInt, batch) || !rows_of(miss_count, device, at::kInt, batch) ||
        (miss_count && miss_count->numel() != batch)) {
        return not_handled();
    }
    const int rc = g_lookup(
        residency_map.data_ptr(), es_map, residency_map.stride(0), residency_map.size(1),
        topk.data_ptr(), es_topk, topk.stride(0),
        lengths ? lengths->data_ptr() : nullptr, es_len,
        batch, k,
        slots->data_ptr<int32_t>(), slots->stride(0),
        reinterpret_cast<uint8_t*>(miss->data_ptr()), miss->stride(0),
        miss_list ? miss_list->data_ptr<int32_t>() : nullptr, miss_list ? miss_list->stride(0) : 0,
        miss_count ? miss_count->data_ptr<int32_t>() : nullptr,
        device, stream_of(device));
    auto opt = [](const std::optional<at::Tensor>& t) { return t ? py::cast(*t) : py::none(); };
    return py::make_tuple(rc == 0 ? 0 : kKernelError, py::cast(*slots), py::cast(*miss), opt(miss_list),
                          opt(miss_count));
}

// Exact Python ints only (bool and int subclasses take the checked path); false
// when an element is not one, overflows int64 or falls outside [lo, hi).
bool int_list(const py::sequence& seq, int64_t lo, int64_t hi, std::vector<int64_t>& out) {
    const size_t n = py::len(seq);
    out.resize(n);
    for (size_t i = 0; i < n; ++i) {
        PyObject* item = PySequence_GetItem(seq.ptr(), static_cast<Py_ssize_t>(i));
        if (!item) {
            PyErr_Clear();
            return false;
        }
        const bool exact = PyLong_CheckExact(item);
        int overflow = 0;
        const long long value = exact ? PyLong_AsLongLongAndOverflow(item, &overflow) : 0;
        Py_DECREF(item);
        if (!exact || overflow || value < lo || value >= hi) {
            PyErr_Clear();
            return false;
        }
        out[i] = value;
    }
    return true;
}

// resolve_shared_block_locations_batched: (status, valid, physical).
py::tuple shared_blocks(const at::Tensor& block_ids, const py::sequence& source_rows, const at::Tensor& seq_len,
                        const py::sequence& shared_tokens, int64_t block_size, const at::Tensor& table,
                        const at::Tensor& mapping, bool exclude_newest, std::optional<at::Tensor> masked) {
    auto not_handled = [] { return py::make_tuple(kNotHandled, py::none(), py::none()); };
    if (!g_shared || block_ids.dim() != 2 || block_size < 1 || block_size > (int64_t{1} << 30) ||
        table.dim() != 2 || table.size(1) == 0 || mapping.dim() != 1 || mapping.numel() == 0 ||
        seq_len.dim() != 1) {
        return not_handled();
    }
    const int64_t requests = block_ids.size(0), per_request = block_ids.size(1);
    const at::Tensor* masked_ptr = masked ? &*masked : nullptr;
    const int device = common_device({&block_ids, &seq_len, &table, &mapping, masked_ptr});
    const int es_blocks = index_size(block_ids), es_len = index_size(seq_len);
    const int es_table = index_size(table), es_map = index_size(mapping);
    if (device < 0 || requests == 0 || per_request == 0 || requests > EKV_SHARED_INLINE_MAX || !es_blocks ||
        !es_len || !es_table || !es_map || seq_len.numel() != requests) {
        return not_handled();
    }
    if (masked && (masked->sizes() != block_ids.sizes() || masked->scalar_type() != block_ids.scalar_type() ||
                   masked->strides() != block_ids.strides())) {
        return not_handled();
    }
    std::vector<int64_t> rows, prefixes;
    if (!int_list(source_rows, 0, table.size(0), rows) ||
        !int_list(shared_tokens, 0, std::numeric_limits<int64_t>::max(), prefixes) ||
        static_cast<int64_t>(rows.size()) != requests || static_cast<int64_t>(prefixes.size()) != requests) {
        return not_handled();
    }
    const auto options = block_ids.options();
    at::Tensor valid = at::empty({requests, per_request}, options.dtype(at::kBool));
    at::Tensor physical = at::empty({requests, per_request, block_size}, options.dtype(at::kInt));
    const int rc = g_shared(
        block_ids.data_ptr(), es_blocks, requests, per_request, block_ids.stride(0), block_ids.stride(1),
        rows.data(), 0, prefixes.data(), 0, seq_len.data_ptr(), es_len, seq_len.stride(0), block_size,
        table.data_ptr(), es_table, table.size(0), table.size(1), table.stride(0), table.stride(1),
        mapping.data_ptr(), es_map, mapping.numel(), mapping.stride(0), 1,
        reinterpret_cast<uint8_t*>(valid.data_ptr()), physical.data_ptr<int32_t>(),
        masked ? masked->data_ptr() : nullptr, exclude_newest ? 1 : 0, device, stream_of(device));
    return py::make_tuple(rc == 0 ? 0 : kKernelError, valid, physical);
}

// Index tensors of a gather: positions [B, S], request_ids / lengths [B], and the
// table / slot offsets the addressing mode uses (mode 0 direct, 1 indirect, 2
// mapped).  Every given tensor CUDA on one device and contiguous (the Python
// API checks the unused table too); element sizes of the used ones in `es`.
struct GatherIndex {
    int device = -1;
    int es[5] = {0, 0, 0, 8, 8};  // positions, request_ids, lengths, table, offsets
    const void* table = nullptr;
    const void* offsets = nullptr;
};

bool gather_index(const at::Tensor& positions, const at::Tensor& request_ids, const at::Tensor& lengths,
                  const std::optional<at::Tensor>& request_table, const std::optional<at::Tensor>& slot_offsets,
                  int mode, GatherIndex& out) {
    const at::Tensor* table = request_table ? &*request_table : nullptr;
    const at::Tensor* offsets = slot_offsets ? &*slot_offsets : nullptr;
    out.device = common_device({&positions, &request_ids, &lengths, table, offsets});
    if (out.device < 0) return false;
    for (const at::Tensor* t : {&positions, &request_ids, &lengths, table, offsets}) {
        if (t && !t->is_contiguous()) return false;
    }
    if ((mode >= 1 && !table) || (mode == 1 && !offsets)) return false;
    out.es[0] = index_size(positions);
    out.es[1] = index_size(request_ids);
    out.es[2] = index_size(lengths);
    if (mode >= 1) {
        out.es[3] = index_size(*table);
        out.table = table->data_ptr();
    }
    if (mode == 1) {
        out.es[4] = index_size(*offsets);
        out.offsets = offsets->data_ptr();
    }
    for (int e : out.es) {
        if (!e) return false;
    }
    return true;
}

bool rows_shape(const at::Tensor& t, int64_t batch, int64_t selected, int64_t width) {
    return t.dim() == 3 && t.size(0) == batch && t.size(1) == selected && t.size(2) == width;
}

// gather_rows (the reference's single-plane call).
int gather_rows(const at::Tensor& raw, const at::Tensor& positions, const at::Tensor& request_ids,
                const at::Tensor& lengths, const std::optional<at::Tensor>& request_table,
                const std::optional<at::Tensor>& slot_offsets, const at::Tensor& output, int64_t width,
                int64_t table_width, int64_t request_stride, int64_t sink_elements, bool indirect) {
    if (!g_gather || positions.dim() != 2) return kNotHandled;
    const int64_t batch = positions.size(0), selected = positions.size(1);
    if (!rows_shape(output, batch, selected, width)) return kNotHandled;
    if (batch == 0 || selected == 0) return 0;  // no-op, as the reference
    const int mode = indirect ? 1 : 0;
    GatherIndex ix;
    if (!gather_index(positions, request_ids, lengths, request_table, slot_offsets, mode, ix)) return kNotHandled;
    if (common_device({&raw, &output}) != ix.device || !raw.is_contiguous() || !output.is_contiguous() ||
        raw.scalar_type() != output.scalar_type()) {
        return kNotHandled;
    }
    const int rc = g_gather(
        raw.data_ptr(), output.data_ptr(), raw.element_size(), positions.data_ptr(), ix.es[0],
        request_ids.data_ptr(), ix.es[1], lengths.data_ptr(), ix.es[2], ix.table, ix.es[3], ix.offsets, ix.es[4],
        batch, selected, width, table_width, request_stride, sink_elements, mode, ix.device, stream_of(ix.device));
    return rc == 0 ? 0 : kKernelError;
}

// gather_rows_planes: one row selection over every plane, EKV_MAX_PLANES planes per launch.
int gather_rows_planes(const std::vector<at::Tensor>& planes, const std::vector<at::Tensor>& outputs,
                       const at::Tensor& positions, const at::Tensor& request_ids, const at::Tensor& lengths,
                       const std::optional<at::Tensor>& request_table,
                       const std::optional<at::Tensor>& slot_offsets, int64_t width, int64_t max_tokens,
                       int64_t request_stride, int64_t sink_elements, bool indirect, bool mapped) {
    if (!g_gather_planes || planes.size() != outputs.size() || positions.dim() != 2 || (indirect && mapped)) {
        return kNotHandled;
    }
    const int64_t batch = positions.size(0), selected = positions.size(1);
    for (const at::Tensor& out : outputs) {
        if (!rows_shape(out, batch, selected, width)) return kNotHandled;
    }
    if (planes.empty() || batch == 0 || selected == 0) return 0;
    const int mode = mapped ? 2 : (indirect ? 1 : 0);
    GatherIndex ix;
    if (!gather_index(positions, request_ids, lengths, request_table, slot_offsets, mode, ix)) return kNotHandled;
    const at::ScalarType dtype = planes[0].scalar_type();
    for (size_t p = 0; p < planes.size(); ++p) {
        const at::Tensor& src = planes[p];
        const at::Tensor& dst = outputs[p];
        if (common_device({&src, &dst}) != ix.device || !src.is_contiguous() || !dst.is_contiguous() ||
            src.scalar_type() != dtype || dst.scalar_type() != dtype) {
            return kNotHandled;
        }
    }
    // A residency map is indexed by token: its row width is the map's, not the layout's.
    const int64_t table_width = mode == 2 ? request_table->size(-1) : max_tokens;
    const int64_t itemsize = planes[0].element_size();
    void* stream = stream_of(ix.device);
    uint64_t src[EKV_MAX_PLANES], dst[EKV_MAX_PLANES];
    for (size_t start = 0; start < planes.size(); start += EKV_MAX_PLANES) {
        const int n = static_cast<int>(std::min<size_t>(EKV_MAX_PLANES, planes.size() - start));
        for (int p = 0; p < n; ++p) {
            src[p] = reinterpret_cast<uint64_t>(planes[start + p].data_ptr());
            dst[p] = reinterpret_cast<uint64_t>(outputs[start + p].data_ptr());
        }
        const int rc = g_gather_planes(
            src, dst, n, itemsize, positions.data_ptr(), ix.es[0], request_ids.data_ptr(), ix.es[1],
            lengths.data_ptr(), ix.es[2], ix.table, ix.es[3], ix.offsets, ix.es[4], batch, selected, width,
            table_width, request_stride, sink_elements, mode, ix.device, stream);
        if (rc != 0) return kKernelError;
    }
    return 0;
}

// ---------------------------------------------------------------- a serving step

const at::Tensor* optional_tensor(const std::optional<at::Tensor>& t) { return t ? &*t : nullptr; }

// Element size of a contiguous one-dimensional index tensor with `count` entries (-1: any), or 0.
int vector_size(const at::Tensor& t, int64_t count) {
    if (t.dim() != 1 || (t.numel() > 1 && t.stride(0) != 1) || (count >= 0 && t.size(0) != count)) return 0;
    return index_size(t);
}

constexpr int64_t kInt32Max = std::numeric_limits<int32_t>::max();

// (status, query_starts, slot_map, positions, lengths, pages_used): fresh outputs.
py::tuple extend_block_tables(const at::Tensor& tables, const at::Tensor& lengths, const at::Tensor& fresh,
                              const at::Tensor& free_pages, int64_t page_size, int64_t max_tokens,
                              const std::optional<at::Tensor>& rows) {
    auto status = [](int rc) { return py::make_tuple(rc, py::none(), py::none(), py::none(), py::none(), py::none()); };
    if (!g_extend || page_size < 1 || page_size > kInt32Max || max_tokens < 0 || max_tokens > kInt32Max) {
        return status(kNotHandled);
    }
    const int device = common_device({&tables, &lengths, &fresh, &free_pages, optional_tensor(rows)});
    if (device < 0 || tables.scalar_type() != at::kInt || free_pages.scalar_type() != at::kInt || tables.dim() != 2 ||
        (tables.size(1) > 1 && tables.stride(1) != 1) || (tables.size(0) > 1 && tables.stride(0) < tables.size(1)) ||
        tables.size(1) > kInt32Max / page_size || lengths.dim() != 1) {
        return status(kNotHandled);
    }
    const int64_t batch = lengths.size(0);
    const int len_es = vector_size(lengths, batch), fresh_es = vector_size(fresh, batch);
    const int rows_es = rows ? vector_size(*rows, batch) : 8;
    if (!len_es || !fresh_es || !rows_es || !vector_size(free_pages, -1)) return status(kNotHandled);
    // Five outputs in one allocation; the views are made without the dispatcher, which took most of the call.
    const at::Tensor flat = at::empty({2 * batch + 2 * max_tokens + 2}, tables.options());
    int64_t offset = 0;
    const auto part = [&](int64_t count) {
        at::Tensor view = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(flat.storage()), flat.key_set(), flat.dtype());
        view.unsafeGetTensorImpl()->set_storage_offset(offset);
        view.unsafeGetTensorImpl()->set_sizes_contiguous({count});
        offset += count;
        return view;
    };
    at::Tensor starts = part(batch + 1), slots = part(max_tokens), positions = part(max_tokens);
    at::Tensor after = part(batch), used = part(1);
    const int rc = g_extend(
        tables.data_ptr<int32_t>(), tables.size(0), tables.size(1), tables.stride(0),
        rows ? rows->data_ptr() : nullptr, rows_es, lengths.data_ptr(), len_es, fresh.data_ptr(), fresh_es, batch,
        free_pages.data_ptr<int32_t>(), free_pages.size(0), page_size, max_tokens, starts.data_ptr<int32_t>(),
        slots.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), after.data_ptr<int32_t>(), used.data_ptr<int32_t>(),
        device, stream_of(device));
    if (rc != 0) return status(kKernelError);
    return py::make_tuple(0, starts, slots, positions, after, used);
}

// Elements between the rows of [count, ...] when each row is contiguous, or -1; `elements` of one row.
int64_t row_stride(const at::Tensor& t, int64_t& elements) {
    elements = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
        if (t.size(d) != 1 && t.stride(d) != elements) return -1;
        elements *= t.size(d);
    }
    return t.size(0) > 1 ? t.stride(0) : elements;
}

int append_rows(const std::vector<at::Tensor>& rows, const at::Tensor& slot_map, const std::vector<at::Tensor>& planes) {
    if (!g_append || rows.size() != planes.size() || planes.size() > EKV_MAX_PLANES || planes.empty()) return kNotHandled;
    const int map_es = vector_size(slot_map, -1);
    if (!map_es || !slot_map.is_cuda()) return kNotHandled;
    const int device = slot_map.get_device();
    const int64_t tokens = slot_map.size(0);
    uint64_t src[EKV_MAX_PLANES], dst[EKV_MAX_PLANES];
    int64_t elements = 0, src_stride = 0, dst_stride = 0;
    const at::ScalarType dtype = planes[0].scalar_type();
    for (size_t i = 0; i < planes.size(); ++i) {
        const at::Tensor& row = rows[i];
        const at::Tensor& plane = planes[i];
        if (common_device({&row, &plane}) != device || row.dim() < 2 || row.size(0) != tokens ||
            row.sizes().slice(1) != plane.sizes().slice(1) || row.scalar_type() != dtype || plane.scalar_type() != dtype ||
            row.sizes() != rows[0].sizes() || plane.sizes() != planes[0].sizes()) {
            return kNotHandled;
        }
        int64_t of_row, of_plane;
        const int64_t from = row_stride(row, of_row), to = row_stride(plane, of_plane);
        if (from < 0 || to < of_plane || (i && (from != src_stride || to != dst_stride))) return kNotHandled;
        elements = of_row;
        src_stride = from;
        dst_stride = to;
        src[i] = reinterpret_cast<uint64_t>(row.data_ptr());
        dst[i] = reinterpret_cast<uint64_t>(plane.data_ptr());
    }
    if (!tokens || !planes[0].size(0) || !elements) return 0;
    const int64_t itemsize = planes[0].element_size();
    const int rc = g_append(src, dst, static_cast<int>(planes.size()), elements * itemsize, src_stride * itemsize,
                            dst_stride * itemsize, slot_map.data_ptr(), map_es, tokens, planes[0].size(0), device,
                            stream_of(device));
    return rc == 0 ? 0 : kKernelError;
}

// [count, heads, dim] with contiguous, 16-byte aligned rows of 16-bit values; `apart`: that do not overlap.
bool head_rows_ok(const at::Tensor& t, bool apart) {
    if (t.stride(2) != 1 || reinterpret_cast<uint64_t>(t.data_ptr()) % 16) return false;
    for (int d = 0; d < 2; ++d) {
        if (t.size(d) > 1 && (t.stride(d) % 8 || (apart && t.stride(d) < t.size(2)))) return false;
    }
    return true;
}

int64_t stride_of(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// Entries of `width` elements, [tokens, heads], of which no two overlap.
bool entries_apart(const at::Tensor& t, int64_t width) {
    const int64_t tokens = t.size(0), heads = t.size(1), token = stride_of(t, 0), head = stride_of(t, 1);
    if ((heads > 1 && head < width) || (tokens > 1 && token < width)) return false;
    return tokens <= 1 || heads <= 1 || token >= (heads - 1) * head + width || head >= (tokens - 1) * token + width;
}

// The addresses a tensor spans; empty for one without elements.
struct Extent {
    int64_t begin = 0, end = 0;
    Extent() = default;
    explicit Extent(const at::Tensor* t) {
        if (!t || !t->numel()) return;
        const at::IntArrayRef sizes = t->sizes(), strides = t->strides();
        int64_t last = 0;
        for (size_t d = 0; d < sizes.size(); ++d) last += (sizes[d] - 1) * strides[d];
        begin = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t->const_data_ptr()));
        end = begin + (last + 1) * static_cast<int64_t>(t->element_size());
    }
    bool meets(const Extent& other) const {
        return begin < end && other.begin < other.end && begin < other.end && other.begin < end;
    }
};

// Whether [tokens, heads(, dim)] tensors share an element: exact where their strides agree, by extents otherwise.
bool collide(const at::Tensor& a, const at::Tensor& b) {
    if (!Extent(&a).meets(Extent(&b))) return false;
    const int64_t size_a = a.element_size(), size_b = b.element_size();
    const int64_t width_a = (a.dim() == 3 ? a.size(2) : 1) * size_a, width_b = (b.dim() == 3 ? b.size(2) : 1) * size_b;
    struct Axis {
        int64_t step, of_a, of_b;
    } axes[2];
    for (int d = 0; d < 2; ++d) {
        const int64_t step_a = a.stride(d) * size_a, step_b = b.stride(d) * size_b;
        if (a.size(d) > 1 && b.size(d) > 1 && step_a != step_b) return true;
        axes[d] = {a.size(d) > 1 ? step_a : (b.size(d) > 1 ? step_b : 0), a.size(d), b.size(d)};
    }
    if (axes[0].step < axes[1].step) std::swap(axes[0], axes[1]);
    const int64_t most[2] = {std::max(axes[0].of_a, axes[0].of_b), std::max(axes[1].of_a, axes[1].of_b)};
    const int64_t width = std::max(width_a, width_b);
    if ((most[1] > 1 && axes[1].step < width) || (most[0] > 1 && axes[0].step < (most[1] - 1) * axes[1].step + width)) {
        return true;
    }
    const int64_t delta = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.data_ptr())) -
                          static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.data_ptr()));
    // Quotients are rounded towards 0 here: one more candidate on the low side.
    const auto first = [](int64_t x, int64_t step) { return step ? x / step - 2 : 0; };
    const auto last = [](int64_t x, int64_t step) { return step ? x / step + 2 : 0; };
    for (int64_t i = first(delta, axes[0].step); i <= last(delta, axes[0].step); ++i) {
        if (i <= -axes[0].of_b || i >= axes[0].of_a) continue;
        const int64_t left = delta - i * axes[0].step;
        for (int64_t j = first(left, axes[1].step); j <= last(left, axes[1].step); ++j) {
            if (j <= -axes[1].of_b || j >= axes[1].of_a) continue;
            const int64_t apart = left - j * axes[1].step;
            if (-width_b < apart && apart < width_a) return true;
        }
    }
    return false;
}

// (status, out, lse or None)
py::tuple shared_prefix_attention(const at::Tensor& query, const at::Tensor& k_plane, const at::Tensor& v_plane,
                                  const at::Tensor& tables, const at::Tensor& lengths, int64_t page_size,
                                  int64_t shared_tokens, int64_t source_row, const std::optional<at::Tensor>& rows,
                                  const std::optional<at::Tensor>& starts, std::optional<double> scale,
                                  std::optional<at::Tensor> out, std::optional<at::Tensor> lse, bool want_lse) {
    auto status = [](int rc) { return py::make_tuple(rc, py::none(), py::none()); };
    const int device = common_device({&query, &k_plane, &v_plane, &tables, &lengths, optional_tensor(rows),
                                      optional_tensor(starts), optional_tensor(out), optional_tensor(lse)});
    if (!g_attention || device < 0 || query.dim() != 3 || k_plane.dim() != 3 || v_plane.sizes() != k_plane.sizes()) {
        return status(kNotHandled);
    }
    const at::ScalarType dtype = query.scalar_type();
    const int64_t tokens = query.size(0), heads = query.size(1), dim = query.size(2);
    const int64_t slots = k_plane.size(0), kv_heads = k_plane.size(1);
    if ((dtype != at::kBFloat16 && dtype != at::kHalf) || k_plane.scalar_type() != dtype || v_plane.scalar_type() != dtype ||
        (dim != 64 && dim != 128) || k_plane.size(2) != dim || !kv_heads || !heads || heads % kv_heads) {
        return status(kNotHandled);
    }
    if (out && (out->scalar_type() != dtype || out->sizes() != query.sizes())) return status(kNotHandled);
    if (!head_rows_ok(query, false) || !head_rows_ok(k_plane, true) || !head_rows_ok(v_plane, true) ||
        (out && (!head_rows_ok(*out, true) || !entries_apart(*out, dim)))) {
        return status(kNotHandled);
    }
    if (lse && (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != tokens || lse->size(1) != heads ||
                !entries_apart(*lse, 1))) {
        return status(kNotHandled);
    }
    if (page_size < 1 || page_size > kInt32Max || tables.dim() != 2 || (tables.size(1) > 1 && tables.stride(1) != 1) ||
        !index_size(tables) || tables.size(1) > (kInt32Max - 255) / page_size || shared_tokens < 0 ||
        shared_tokens > tables.size(1) * page_size ||
        (shared_tokens && (source_row < 0 || source_row >= tables.size(0))) || lengths.dim() != 1) {
        return status(kNotHandled);
    }
    const int64_t batch = lengths.size(0);
    const int len_es = vector_size(lengths, batch), rows_es = rows ? vector_size(*rows, batch) : 8;
    const int starts_es = starts ? vector_size(*starts, batch + 1) : 8;
    if (!len_es || !rows_es || !starts_es || (!starts && tokens != batch) || tokens * heads > kInt32Max ||
        batch + (tokens * heads / kv_heads + 255) / 256 > EKV_ATTENTION_MAX_ROW_TILES) {
        return status(kNotHandled);
    }
    if (out || lse) {
        // Extents first: the exact answer is needed only where they meet.
        const Extent results[2] = {Extent(optional_tensor(out)), Extent(optional_tensor(lse))};
        for (const at::Tensor* read : {&query, &k_plane, &v_plane}) {
            const Extent its(read);
            if (lse && results[1].meets(its) && collide(*lse, *read)) return status(kNotHandled);
            if (!out || !results[0].meets(its)) continue;
            const bool query_itself = read == &query && out->const_data_ptr() == query.const_data_ptr() &&
                                      stride_of(*out, 0) == stride_of(query, 0) && stride_of(*out, 1) == stride_of(query, 1);
            if (!query_itself && collide(*out, *read)) return status(kNotHandled);
        }
        for (const at::Tensor* read : {&tables, &lengths, optional_tensor(rows), optional_tensor(starts)}) {
            const Extent its(read);
            if (results[0].meets(its) || results[1].meets(its)) return status(kNotHandled);
        }
        if (out && lse && results[0].meets(results[1]) && collide(*out, *lse)) return status(kNotHandled);
    }
    const double factor = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(dim));
    if (!(factor >= 1.5e-45 && factor <= 2.3e38)) return status(kNotHandled);
    if (!out) out = at::empty(query.sizes(), query.options());
    if (!lse && want_lse) lse = at::empty({tokens, heads}, query.options().dtype(at::kFloat));
    int64_t bytes = 0;
    if (g_workspace(tokens, batch, static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(dim), device, &bytes)) {
        return status(kKernelError);
    }
    const at::Tensor workspace = at::empty({bytes}, query.options().dtype(at::kByte));
    const int rc = g_attention(
        query.data_ptr(), stride_of(query, 0), stride_of(query, 1), k_plane.data_ptr(), stride_of(k_plane, 0),
        stride_of(k_plane, 1), v_plane.data_ptr(), stride_of(v_plane, 0), stride_of(v_plane, 1), slots,
        dtype == at::kBFloat16 ? EKV_BF16 : EKV_FP16, static_cast<int>(dim), static_cast<int>(heads),
        static_cast<int>(kv_heads), tokens, batch, tables.data_ptr(), index_size(tables), tables.size(0), tables.size(1),
        tables.stride(0), page_size, rows ? rows->data_ptr() : nullptr, rows_es, lengths.data_ptr(), len_es,
        starts ? starts->data_ptr() : nullptr, starts_es, shared_tokens, source_row, static_cast<float>(factor),
        out->data_ptr(), stride_of(*out, 0), stride_of(*out, 1), lse ? lse->data_ptr<float>() : nullptr,
        lse ? lse->stride(0) : 0, lse ? lse->stride(1) : 0, workspace.data_ptr(), bytes, device, stream_of(device));
    if (rc != 0) return status(kKernelError);
    return py::make_tuple(0, *out, lse ? py::cast(*lse) : py::object(py::none()));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "Compiled binding of the per-call residency lookups of libekv_b200.so";
    m.def("bind", &bind, "set the addresses of the C entry points");
    m.def("resolve_resident", &resolve_resident);
    m.def("lookup_slots", &lookup_slots, py::arg("residency_map"), py::arg("topk"), py::arg("lengths"),
          py::arg("slots"), py::arg("miss"), py::arg("miss_list"), py::arg("miss_count"), py::arg("compact"));
    m.def("shared_blocks", &shared_blocks);
    m.def("gather_rows", &gather_rows);
    m.def("gather_rows_planes", &gather_rows_planes);
    m.def("extend_block_tables", &extend_block_tables);
    m.def("append_rows", &append_rows);
    m.def("shared_prefix_attention", &shared_prefix_attention);
    m.def("collide", &collide);
    m.attr("NOT_HANDLED") = kNotHandled;
    m.attr("KERNEL_ERROR") = kKernelError;
}
