// Block tables, slot maps and the row append of a serving step.
//
// extend_tables_kernel.  Request b holds L tokens and gains n; with page size p it
// needs  ceil((L + n) / p) - ceil(L / p)  pages.  With T(b) and P(b) the inclusive
// sums of tokens and pages over the batch, requests are granted while T(b) <= N
// (slot-map capacity) and P(b) <= F (pages offered); both sums grow with b, so the
// granted requests are a prefix of the batch and one scan decides everything.  The
// granted request's pages are free_pages[P(b-1) .. P(b)), and its i-th token (position
// L + i) has slot  page(position / p) * p + position % p.
// Bound by latency up to ~10^5 tokens: one launch in which EVERY block scans the
// whole batch (1024 requests a pass; two dependent 4-byte loads and one block scan)
// and then places only its own slice of tokens and pages, so no second launch or
// grid-wide wait separates the scan from the placement: 6.3 us on the device for 8
// requests, 8.4 us for 1024 requests of one token or 257,000 tokens of prompts; 13 us a
// call from Python, which binds it.
//
// append_rows_kernel.  plane[slot_map[i]] = row[i] for every plane: HBM-bound, one
// read and one write of each row.  Rows are flattened to vectors (plane in grid.y) and
// each thread keeps kAppendUnroll independent copies in flight: 65,536 tokens of 2 KB in K
// and in V, one in 97 skipped, 84 us, 0.96 of the measured copy peak; 64 tokens 4.2 us (9 us a call).
#include "common.cuh"

namespace ekv {
namespace {

constexpr int kTableThreads = 1024;
constexpr int kTableWarps = kTableThreads / 32;
// Tokens (and pages) one block places.
constexpr int kTokensPerBlock = 2 * kTableThreads;

struct TableParams {
    int32_t* tables;
    const void* rows;  // null: request b is table row b
    const void* lengths;
    const void* fresh;
    const int32_t* free_pages;
    int32_t* starts;
    int32_t* slot_map;
    int32_t* positions;
    int32_t* lengths_out;
    int32_t* pages_used;
    int64_t table_rows, table_width, table_stride;
    int64_t batch, n_free, capacity;
    int64_t page_size;
    int64_t slice;  // tokens (and pages) of one block
    int rows_es, len_es, fresh_es;
    int page_log2;  // -1: page_size is not a power of two
};

__device__ __forceinline__ uint32_t page_of(const TableParams& p, uint32_t position) {
    return p.page_log2 >= 0 ? position >> p.page_log2 : position / static_cast<uint32_t>(p.page_size);
}

// Inclusive scan of (a, b) over the block; totals of the block in (ta, tb).
static_assert(kTableWarps == 32, "a lane per warp");
__device__ __forceinline__ void block_scan(int64_t& a, int64_t& b, int64_t& ta, int64_t& tb, int64_t (*sums)[2]) {
    const unsigned lane = lane_id(), warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t ua = __shfl_up_sync(0xffffffffu, a, d), ub = __shfl_up_sync(0xffffffffu, b, d);
        if (lane >= d) a += ua, b += ub;
    }
    if (lane == 31) sums[warp][0] = a, sums[warp][1] = b;
    __syncthreads();
    // Every warp scans the warps' sums, a lane each.
    int64_t ra = sums[lane][0], rb = sums[lane][1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t ua = __shfl_up_sync(0xffffffffu, ra, d), ub = __shfl_up_sync(0xffffffffu, rb, d);
        if (lane >= d) ra += ua, rb += ub;
    }
    ta = __shfl_sync(0xffffffffu, ra, 31);
    tb = __shfl_sync(0xffffffffu, rb, 31);
    const int64_t before_a = __shfl_sync(0xffffffffu, ra, warp - 1), before_b = __shfl_sync(0xffffffffu, rb, warp - 1);
    if (warp) a += before_a, b += before_b;
}

// Largest i in [0, count) with start[i] <= x, for start[0] <= x (start ascending).
__device__ __forceinline__ int last_at_most(const int64_t* start, int count, int64_t x) {
    int low = 0, high = count;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (start[mid] <= x) {
            low = mid;
        } else {
            high = mid;
        }
    }
    return low;
}

__global__ void __launch_bounds__(kTableThreads) extend_tables_kernel(const __grid_constant__ TableParams p) {
    __shared__ int64_t sums[kTableWarps][2];
    __shared__ int64_t token_start[kTableThreads], page_start[kTableThreads];
    __shared__ int64_t row_of[kTableThreads];
    __shared__ uint32_t held_of[kTableThreads], had_of[kTableThreads];
    grid_dependency_wait();
    allow_dependents();
    const int64_t begin = blockIdx.x * p.slice;
    const int64_t end = begin + p.slice < p.capacity ? begin + p.slice : p.capacity;
    const int64_t page_end = begin + p.slice;  // pages: the last block takes what is left
    int64_t tokens_before = 0, pages_before = 0;
    bool open = true;
    for (int64_t first = 0; first < p.batch; first += kTableThreads) {
        const int64_t b = first + threadIdx.x;
        int64_t held = 0, fresh = 0, row = -1;
        if (b < p.batch) {
            held = load_index(p.lengths, p.len_es, b);
            fresh = load_index(p.fresh, p.fresh_es, b);
            row = p.rows ? load_index(p.rows, p.rows_es, b) : b;
            if (held < 0) held = 0;
        }
        // Compared in this order nothing overflows: room is at most 2^31.
        const int64_t room = p.table_width * p.page_size;
        const bool active = open && row >= 0 && row < p.table_rows && fresh > 0 && held <= room && fresh <= room - held;
        const uint32_t had = active ? static_cast<uint32_t>((held + p.page_size - 1) / p.page_size) : 0;
        int64_t tokens = active ? fresh : 0;
        int64_t pages = active ? (held + fresh + p.page_size - 1) / p.page_size - had : 0;
        const int64_t own_tokens = tokens, own_pages = pages;
        int64_t tile_tokens, tile_pages;
        block_scan(tokens, pages, tile_tokens, tile_pages, sums);
        const bool fits = active && tokens_before + tokens <= p.capacity && pages_before + pages <= p.n_free;
        // Everything after the first request that does not fit gets nothing.
        const bool closed = __syncthreads_or(active && !fits);
        if (closed) {
            int64_t granted_tokens = fits ? own_tokens : 0, granted_pages = fits ? own_pages : 0;
            block_scan(granted_tokens, granted_pages, tile_tokens, tile_pages, sums);
            tokens = granted_tokens;
            pages = granted_pages;
        }
        const int64_t my_tokens = fits ? own_tokens : 0, my_pages = fits ? own_pages : 0;
        token_start[threadIdx.x] = tokens_before + tokens - my_tokens;
        page_start[threadIdx.x] = pages_before + pages - my_pages;
        row_of[threadIdx.x] = row;
        held_of[threadIdx.x] = static_cast<uint32_t>(held);
        had_of[threadIdx.x] = had;
        if (blockIdx.x == 0 && b < p.batch) {
            p.starts[b] = static_cast<int32_t>(tokens_before + tokens - my_tokens);
            // A length that 32 bits do not hold (never granted) is kept at their largest value.
            const int64_t after = held + my_tokens;
            p.lengths_out[b] = static_cast<int32_t>(after < INT32_MAX ? after : INT32_MAX);
        }
        __syncthreads();
        const int count = static_cast<int>(p.batch - first < kTableThreads ? p.batch - first : kTableThreads);
        // This tile's tokens inside the block's slice.
        const int64_t token_high = tokens_before + tile_tokens < end ? tokens_before + tile_tokens : end;
        for (int64_t t = (tokens_before > begin ? tokens_before : begin) + threadIdx.x; t < token_high;
             t += kTableThreads) {
            const int r = last_at_most(token_start, count, t);
            const uint32_t position = held_of[r] + static_cast<uint32_t>(t - token_start[r]);
            const uint32_t index = page_of(p, position);
            const int32_t page = index < had_of[r]
                                     ? p.tables[row_of[r] * p.table_stride + index]
                                     : p.free_pages[page_start[r] + (index - had_of[r])];
            const int64_t slot = static_cast<int64_t>(page) * p.page_size + (position - index * static_cast<uint32_t>(p.page_size));
            p.slot_map[t] = page >= 0 && slot <= INT32_MAX ? static_cast<int32_t>(slot) : -1;
            p.positions[t] = static_cast<int32_t>(position);
        }
        // This tile's new table entries: page k belongs to the block whose slice holds k.
        const int64_t all_pages = pages_before + tile_pages;
        const int64_t page_high = blockIdx.x + 1 == gridDim.x || all_pages < page_end ? all_pages : page_end;
        for (int64_t k = (pages_before > begin ? pages_before : begin) + threadIdx.x; k < page_high;
             k += kTableThreads) {
            const int r = last_at_most(page_start, count, k);
            p.tables[row_of[r] * p.table_stride + had_of[r] + (k - page_start[r])] = p.free_pages[k];
        }
        tokens_before += tile_tokens;
        pages_before += tile_pages;
        open = open && !closed;  // a pass behind the closing one grants nothing, so none in it is refused
        __syncthreads();
    }
    for (int64_t t = (tokens_before > begin ? tokens_before : begin) + threadIdx.x; t < end; t += kTableThreads) {
        p.slot_map[t] = -1;
        p.positions[t] = -1;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.starts[p.batch] = static_cast<int32_t>(tokens_before);
        *p.pages_used = static_cast<int32_t>(pages_before);
    }
}

constexpr int kAppendThreads = 256;
constexpr int kAppendUnroll = 4;

struct AppendParams {
    uint64_t src[EKV_MAX_PLANES];
    uint64_t dst[EKV_MAX_PLANES];
    const void* slot_map;
    int64_t tokens, slots;
    int64_t src_stride, dst_stride;  // bytes
    int64_t vectors;                 // vectors of one row
    int vector_log2;                 // -1: not a power of two
    int map_es;
};

template <typename Vector>
__global__ void __launch_bounds__(kAppendThreads) append_rows_kernel(const __grid_constant__ AppendParams p) {
    grid_dependency_wait();
    allow_dependents();
    const char* src = reinterpret_cast<const char*>(p.src[blockIdx.y]);
    char* dst = reinterpret_cast<char*>(p.dst[blockIdx.y]);
    const int64_t total = p.tokens * p.vectors;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kAppendThreads * kAppendUnroll;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kAppendThreads * kAppendUnroll + threadIdx.x; base < total;
         base += step) {
        Vector value[kAppendUnroll];
        char* target[kAppendUnroll];
#pragma unroll
        for (int u = 0; u < kAppendUnroll; ++u) {
            const int64_t item = base + u * kAppendThreads;
            target[u] = nullptr;
            if (item >= total) continue;
            const int64_t token = p.vector_log2 >= 0 ? item >> p.vector_log2 : item / p.vectors;
            const int64_t offset = (item - token * p.vectors) * static_cast<int64_t>(sizeof(Vector));
            const int64_t slot = load_index(p.slot_map, p.map_es, token);
            if (slot < 0 || slot >= p.slots) continue;
            target[u] = dst + slot * p.dst_stride + offset;
            value[u] = __ldcs(reinterpret_cast<const Vector*>(src + token * p.src_stride + offset));
        }
#pragma unroll
        for (int u = 0; u < kAppendUnroll; ++u) {
            if (target[u]) *reinterpret_cast<Vector*>(target[u]) = value[u];
        }
    }
}

template <typename Vector>
void launch_append(AppendParams& p, int n_planes, int64_t row_bytes, int device, cudaStream_t stream) {
    p.vectors = row_bytes / static_cast<int64_t>(sizeof(Vector));
    p.vector_log2 = -1;
    for (int bit = 0; bit < 40; ++bit) {
        if (p.vectors == int64_t{1} << bit) p.vector_log2 = bit;
    }
    const int64_t per_block = kAppendThreads * kAppendUnroll;
    const int64_t wanted = (p.tokens * p.vectors + per_block - 1) / per_block;
    const int64_t cap = int64_t{1} << 20;
    const dim3 grid(static_cast<unsigned>(wanted < cap ? wanted : cap), static_cast<unsigned>(n_planes));
    launch_dependent(append_rows_kernel<Vector>, grid, dim3(kAppendThreads), 0, stream, "append_rows launch", p);
}

}  // namespace
}  // namespace ekv

extern "C" int ekv_extend_block_tables(
    int32_t* block_tables, int64_t table_rows, int64_t table_width, int64_t table_row_stride,
    const void* rows, int rows_esize, const void* lengths, int lengths_esize,
    const void* new_tokens, int new_esize, int64_t batch,
    const int32_t* free_pages, int64_t n_free, int64_t page_size, int64_t max_tokens,
    int32_t* query_starts, int32_t* slot_map, int32_t* positions, int32_t* new_lengths, int32_t* pages_used,
    int device, void* stream) {
    using namespace ekv;
    return guarded([&] {
        require(batch >= 0 && n_free >= 0 && max_tokens >= 0 && table_rows >= 0 && table_width >= 0,
                "negative block-table dimensions");
        require(page_size >= 1 && page_size <= INT32_MAX, "page_size outside [1, 2^31)");
        require(table_width <= INT32_MAX / page_size, "a table row covers more than 2^31 - 1 positions");
        require(max_tokens <= INT32_MAX && n_free <= INT32_MAX, "more than 2^31 - 1 tokens or pages");
        require(query_starts && pages_used, "null pointer argument");
        require(!batch || (lengths && new_tokens && new_lengths && (block_tables || !table_rows || !table_width)),
                "null pointer argument");
        require(!max_tokens || (slot_map && positions), "null pointer argument");
        require(!n_free || free_pages, "null pointer argument");
        if (rows) check_esize(rows_esize, "rows");
        check_esize(lengths_esize, "lengths");
        check_esize(new_esize, "new_tokens");
        bind_device(device);
        TableParams p{};
        p.tables = block_tables;
        p.rows = rows;
        p.lengths = lengths;
        p.fresh = new_tokens;
        p.free_pages = free_pages;
        p.starts = query_starts;
        p.slot_map = slot_map;
        p.positions = positions;
        p.lengths_out = new_lengths;
        p.pages_used = pages_used;
        p.table_rows = table_rows;
        p.table_width = table_width;
        p.table_stride = table_row_stride;
        p.batch = batch;
        p.n_free = n_free;
        p.capacity = max_tokens;
        p.page_size = page_size;
        p.rows_es = rows_esize;
        p.len_es = lengths_esize;
        p.fresh_es = new_esize;
        p.page_log2 = -1;
        for (int bit = 0; bit < 31; ++bit) {
            if (page_size == int64_t{1} << bit) p.page_log2 = bit;
        }
        const int64_t wanted = (max_tokens + kTokensPerBlock - 1) / kTokensPerBlock;
        const int64_t cap = sm_count(device);
        const int64_t grid = wanted < 1 ? 1 : (wanted < cap ? wanted : cap);
        p.slice = (max_tokens + grid - 1) / grid;
        launch_dependent(extend_tables_kernel, dim3(static_cast<unsigned>(grid)), dim3(kTableThreads), 0,
                         static_cast<cudaStream_t>(stream), "extend_block_tables launch", p);
        check_launch("extend_block_tables launch");
    });
}

extern "C" int ekv_append_rows(
    const uint64_t* src, const uint64_t* dst, int n_planes, int64_t row_bytes, int64_t src_row_stride_bytes,
    int64_t dst_row_stride_bytes, const void* slot_map, int map_esize, int64_t tokens, int64_t slots,
    int device, void* stream) {
    using namespace ekv;
    return guarded([&] {
        require(n_planes >= 0 && n_planes <= EKV_MAX_PLANES, "plane count outside [0, EKV_MAX_PLANES]");
        require(tokens >= 0 && slots >= 0 && row_bytes >= 0, "negative row dimensions");
        if (!n_planes || !tokens || !slots || !row_bytes) return;
        require(src && dst && slot_map, "null pointer argument");
        check_esize(map_esize, "slot_map");
        bind_device(device);
        AppendParams p{};
        uint64_t bits = static_cast<uint64_t>(row_bytes) | static_cast<uint64_t>(src_row_stride_bytes) |
                        static_cast<uint64_t>(dst_row_stride_bytes);
        for (int i = 0; i < n_planes; ++i) {
            require(src[i] && dst[i], "null plane address");
            p.src[i] = src[i];
            p.dst[i] = dst[i];
            bits |= src[i] | dst[i];
        }
        p.slot_map = slot_map;
        p.map_es = map_esize;
        p.tokens = tokens;
        p.slots = slots;
        p.src_stride = src_row_stride_bytes;
        p.dst_stride = dst_row_stride_bytes;
        const auto cstream = static_cast<cudaStream_t>(stream);
        // The widest vector that divides every address, stride and the row.
        if (bits % 16 == 0) {
            launch_append<uint4>(p, n_planes, row_bytes, device, cstream);
        } else if (bits % 4 == 0) {
            launch_append<uint32_t>(p, n_planes, row_bytes, device, cstream);
        } else if (bits % 2 == 0) {
            launch_append<uint16_t>(p, n_planes, row_bytes, device, cstream);
        } else {
            launch_append<uint8_t>(p, n_planes, row_bytes, device, cstream);
        }
        check_launch("append_rows launch");
    });
}
