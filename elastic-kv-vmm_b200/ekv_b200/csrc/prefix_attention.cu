// Attention of a batch whose requests share a prefix.
//
// Query token n belongs to request b (query_starts) as its i-th of n_b new tokens and
// sees the tokens j < vis = length_b - n_b + i + 1.  Token j < P is read through the
// source request's table row, every other through the request's own:
//     o = sum_j exp(scale q.k_j) v_j / sum_j exp(scale q.k_j),   lse = log sum_j exp(scale q.k_j).
//
// prefix_rows_kernel: one warp per (token, query head) walks its tokens in order with a
// running maximum and sum in 32 bits (one pass over K and V); the head dimension is
// spread over the lanes, a score is one warp reduction.
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ekv {
namespace {

struct AttentionParams {
    const void* query;
    const void* k_plane;
    const void* v_plane;
    void* out;
    float* lse;  // may be null
    const void* tables;
    const void* rows;    // null: request b is table row b
    const void* lengths;
    const void* starts;  // null: token b is request b's only one
    int64_t q_token, q_head, k_slot, k_head, v_slot, v_head, o_token, o_head, lse_token, lse_head;
    int64_t slots, table_rows, table_width, table_stride, page_size;
    int64_t tokens, batch, shared, source_row;
    int query_heads, group;
    int table_es, rows_es, len_es, starts_es;
    float scale_log2;  // scale * log2(e)
};

// Request of query token n, with the tokens that n sees; false for a token of no request.
__device__ __forceinline__ bool request_of(const AttentionParams& p, int64_t n, int64_t& b, int64_t& seen) {
    int64_t fresh = 1, at = 0;
    b = n;
    if (p.starts) {
        int64_t low = 0, high = p.batch + 1;
        while (high - low > 1) {
            const int64_t mid = (low + high) >> 1;
            if (load_index(p.starts, p.starts_es, mid) <= n) {
                low = mid;
            } else {
                high = mid;
            }
        }
        if (low >= p.batch) return false;
        const int64_t begin = load_index(p.starts, p.starts_es, low), end = load_index(p.starts, p.starts_es, low + 1);
        if (n < begin || n >= end) return false;
        b = low;
        fresh = end - begin;
        at = n - begin;
    }
    seen = load_index(p.lengths, p.len_es, b) - fresh + at + 1;
    return true;
}

// Slot of token j of table row `row`, or -1 where the table has none inside the planes.
__device__ __forceinline__ int64_t slot_of(const AttentionParams& p, int64_t row, int64_t j) {
    if (row < 0 || row >= p.table_rows) return -1;
    const int64_t index = j / p.page_size;
    if (index >= p.table_width) return -1;
    const int64_t page = load_index(p.tables, p.table_es, row * p.table_stride + index);
    if (page < 0 || page >= p.slots) return -1;
    const int64_t slot = page * p.page_size + (j - index * p.page_size);
    return slot < p.slots ? slot : -1;
}

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float x, __half& y) { y = __float2half_rn(x); }

template <typename T, int kDim>
__global__ void __launch_bounds__(128) prefix_rows_kernel(const __grid_constant__ AttentionParams p) {
    constexpr int kPer = kDim / 32;
    grid_dependency_wait();
    allow_dependents();
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int64_t n = item / p.query_heads;
    const int head = static_cast<int>(item - n * p.query_heads);
    const unsigned lane = lane_id();
    int64_t b, seen;
    if (n >= p.tokens || !request_of(p, n, b, seen)) return;
    const int64_t row = p.rows ? load_index(p.rows, p.rows_es, b) : b;
    const int kv_head = head / p.group;
    const T* q = static_cast<const T*>(p.query) + n * p.q_token + head * p.q_head;
    const T* k = static_cast<const T*>(p.k_plane) + kv_head * p.k_head;
    const T* v = static_cast<const T*>(p.v_plane) + kv_head * p.v_head;
    float query[kPer], acc[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        query[i] = to_float(q[lane + 32 * i]);
        acc[i] = 0.f;
    }
    float top = -INFINITY, total = 0.f;
    for (int64_t j = 0; j < seen; ++j) {
        const int64_t slot = slot_of(p, j < p.shared ? p.source_row : row, j);
        if (slot < 0) {
            if (j / p.page_size >= p.table_width) break;
            continue;
        }
        float score = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) score = fmaf(query[i], to_float(k[slot * p.k_slot + lane + 32 * i]), score);
#pragma unroll
        for (int d = 16; d; d >>= 1) score += __shfl_xor_sync(0xffffffffu, score, d);
        score *= p.scale_log2;
        const float higher = fmaxf(top, score);
        const float rescale = top == -INFINITY ? 0.f : exp2f(top - higher);
        const float weight = higher == -INFINITY ? 0.f : exp2f(score - higher);
        top = higher;
        total = total * rescale + weight;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            acc[i] = fmaf(weight, to_float(v[slot * p.v_slot + lane + 32 * i]), acc[i] * rescale);
        }
    }
    T* o = static_cast<T*>(p.out) + n * p.o_token + head * p.o_head;
#pragma unroll
    for (int i = 0; i < kPer; ++i) from_float(total == 0.f ? 0.f : acc[i] / total, o[lane + 32 * i]);
    if (p.lse && lane == 0) {
        p.lse[n * p.lse_token + head * p.lse_head] =
            total == 0.f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
    }
}

template <typename T, int kDim>
void launch_rows(const AttentionParams& p, cudaStream_t stream) {
    const int64_t items = p.tokens * p.query_heads;
    const int64_t grid = (items + 3) / 4;
    require(grid <= INT32_MAX, "too many query rows");
    launch_dependent(prefix_rows_kernel<T, kDim>, dim3(static_cast<unsigned>(grid)), dim3(128), 0, stream,
                     "shared_prefix_attention launch", p);
}

}  // namespace
}  // namespace ekv

extern "C" int ekv_shared_prefix_workspace(int64_t tokens, int64_t batch, int query_heads, int kv_heads, int head_dim,
                                           int device, int64_t* bytes) {
    using namespace ekv;
    return guarded([&] {
        require(bytes != nullptr, "null pointer argument");
        require(tokens >= 0 && batch >= 0 && query_heads >= 0 && kv_heads >= 0, "negative attention dimensions");
        (void)head_dim;
        (void)device;
        *bytes = 0;
    });
}

extern "C" int ekv_shared_prefix_attention(
    const void* query, int64_t q_token_stride, int64_t q_head_stride,
    const void* k_plane, int64_t k_slot_stride, int64_t k_head_stride,
    const void* v_plane, int64_t v_slot_stride, int64_t v_head_stride, int64_t slots,
    int dtype, int head_dim, int query_heads, int kv_heads, int64_t tokens, int64_t batch,
    const void* block_tables, int table_esize, int64_t table_rows, int64_t table_width, int64_t table_row_stride,
    int64_t page_size, const void* rows, int rows_esize, const void* lengths, int lengths_esize,
    const void* query_starts, int starts_esize, int64_t shared_tokens, int64_t source_row, float scale,
    void* out, int64_t o_token_stride, int64_t o_head_stride,
    float* lse, int64_t lse_token_stride, int64_t lse_head_stride,
    void* workspace, int64_t workspace_bytes, int device, void* stream) {
    using namespace ekv;
    return guarded([&] {
        require(tokens >= 0 && batch >= 0 && slots >= 0 && table_rows >= 0 && table_width >= 0,
                "negative attention dimensions");
        require(dtype == EKV_BF16 || dtype == EKV_FP16, "dtype must be EKV_BF16 or EKV_FP16");
        require(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
        require(kv_heads >= 1 && query_heads >= 1 && query_heads % kv_heads == 0,
                "query_heads must be a positive multiple of kv_heads");
        require(page_size >= 1 && page_size <= INT32_MAX, "page_size outside [1, 2^31)");
        require(shared_tokens >= 0 && shared_tokens <= table_width * page_size,
                "shared_tokens outside the table's positions");
        require(!shared_tokens || (source_row >= 0 && source_row < table_rows), "source row is outside the block table");
        require(scale > 0.f && scale <= 3.4e38f, "scale must be positive and finite");
        require(query_starts || tokens == batch, "without query_starts every request has one query token");
        if (!tokens || !batch) return;
        require(query && out && lengths && (block_tables || !table_rows || !table_width) &&
                    ((k_plane && v_plane) || !slots), "null pointer argument");
        const uint64_t bits = reinterpret_cast<uint64_t>(query) | reinterpret_cast<uint64_t>(k_plane) |
                              reinterpret_cast<uint64_t>(v_plane) | reinterpret_cast<uint64_t>(out) |
                              static_cast<uint64_t>((q_token_stride | q_head_stride | k_slot_stride | k_head_stride |
                                                     v_slot_stride | v_head_stride | o_token_stride | o_head_stride) * 2);
        require(bits % 16 == 0, "query, planes and out need 16-byte aligned rows");
        check_esize(table_esize, "block_tables");
        if (rows) check_esize(rows_esize, "rows");
        check_esize(lengths_esize, "lengths");
        if (query_starts) check_esize(starts_esize, "query_starts");
        (void)workspace;
        (void)workspace_bytes;
        bind_device(device);
        AttentionParams p{};
        p.query = query;
        p.k_plane = k_plane;
        p.v_plane = v_plane;
        p.out = out;
        p.lse = lse;
        p.tables = block_tables;
        p.rows = rows;
        p.lengths = lengths;
        p.starts = query_starts;
        p.q_token = q_token_stride;
        p.q_head = q_head_stride;
        p.k_slot = k_slot_stride;
        p.k_head = k_head_stride;
        p.v_slot = v_slot_stride;
        p.v_head = v_head_stride;
        p.o_token = o_token_stride;
        p.o_head = o_head_stride;
        p.lse_token = lse_token_stride;
        p.lse_head = lse_head_stride;
        p.slots = slots;
        p.table_rows = table_rows;
        p.table_width = table_width;
        p.table_stride = table_row_stride;
        p.page_size = page_size;
        p.tokens = tokens;
        p.batch = batch;
        p.shared = shared_tokens;
        p.source_row = source_row;
        p.query_heads = query_heads;
        p.group = query_heads / kv_heads;
        p.table_es = table_esize;
        p.rows_es = rows_esize;
        p.len_es = lengths_esize;
        p.starts_es = starts_esize;
        p.scale_log2 = scale * 1.4426950408889634f;
        const auto cstream = static_cast<cudaStream_t>(stream);
        if (dtype == EKV_BF16) {
            head_dim == 128 ? launch_rows<__nv_bfloat16, 128>(p, cstream) : launch_rows<__nv_bfloat16, 64>(p, cstream);
        } else {
            head_dim == 128 ? launch_rows<__half, 128>(p, cstream) : launch_rows<__half, 64>(p, cstream);
        }
        check_launch("shared_prefix_attention launch");
    });
}
