// Attention of a batch whose requests share a prefix.
//
// Query token n belongs to request b (query_starts) as its i-th of n_b new tokens and
// sees the tokens j < vis = length_b - n_b + i + 1.  Token j < P is read through the
// source request's table row, every other through the request's own:
//     o = sum_j exp(scale q.k_j) v_j / sum_j exp(scale q.k_j),   lse = log sum_j exp(scale q.k_j).
//
// Three kernels.  rows_kernel takes the requests of up to 16 query rows a KV head (a decode step), each
// against its own positions from P on, and a short prefix of a small batch: too few rows for a
// tensor-core tile, so HBM bounds it.  attention_kernel takes the rest: all rows of the batch against the
// shared positions, a matrix product that grows with the batch, and the own positions of requests
// with more rows (prompts).  combine_kernel joins what they leave.  The first two run side by side, each on
// SMs of its own: blocks of attention_kernel that the plan has no work for leave at once.
//
// Work is a list of ITEMS, one per KV head and row tile (up to 256 query rows that read the same
// keys, a row being a token and one of the head's query heads), each a run of 128-position
// tiles.  An item costs a start and so much a tile; the total is cut into one equal share per block,
// so an item may be spread over several, each of which leaves a part (maximum, sum and unscaled output
// in 32 bits).  Every block derives its share from the lengths by itself (one scan over the
// requests), so lengths may change under a captured graph and nothing is read back.
//
// attention_kernel, one tile: S = Q K^T and O += P V on the tensor cores (tcgen05, 128 rows, 32-bit sums
// in tensor memory), a softmax thread per row between them.  The two halves (64 positions) of a tile
// follow one another: the softmax of one runs beside the second product of the other and, right behind it, the first
// product of that half of the next tile, whose scores take the place of its weights.  (A first product of 64
// columns runs at half the tensor cores' rate, since its 128 rows come from shared memory each time; waiting
// for products of whole tiles cost more where the two were compared: 8 requests of up to 400 new tokens over 8001
// shared ones 372 us against 343.)
// Roles by warp: 0-3 and 4-7 softmax of the halves ("slots") 0 and 1 of a row tile; 8-11 copy the K rows,
// 12-15 the V rows into swizzled shared memory (cp.async, 16 bytes a lane, whole rows; slots resolved
// through the table, zeros for positions without one); 16 and 17 issue the products of slots 0 and 1
// (a thread each, so that the waits and commits of one fall beside the other's products); 18 and 19
// pass on the V and K rows that have landed, with the fence between ordinary writes and the tensor cores'
// reads; 18 also walks the block's items and hands them to the others through a small ring.  The queries
// are copied by the softmax warps, as soon as their last product with the ones before is complete.
// An item of more than 128 rows uses both slots on the same K and V (kBoth); a smaller one with many
// tiles gives its even tiles to one slot and its odd ones to the other (kPair; the two join before
// they are written); with few tiles, items alternate between the slots (kSingle).
// What bounds it: no single unit.  Tensor cores (half of whose work runs at half rate), exponential unit and issue
// slots, which eight copying warps share, are each busy 40 to 47 % of the time; the rest is each half waiting for the
// chain of product, softmax and product.  256 requests of 64 heads over 32768 shared tokens and up to 900 own ones:
// 373 us in graph replays for 279 GFLOP, 0.44 of the measured matrix peak.
//
// The maximum a row's weights refer to is raised only when the scores' maximum passes it by 2^8
// (kRaise), which makes rescaling O rare; weights are then at most 2^8.  They are rounded to the 16-bit type
// for the second product (its operand type); the row sum is taken of the unrounded ones.  fp16 holds nothing below
// 2^-25, so its weights are 2^7 times as large (kShift), at most 2^15: what is lost of a long flat tail is then below
// 2^-32 of the maximum's weight.  Sums and outputs carry the factor up to the join, where it cancels.
#include "tensor.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace ekv {
namespace {

constexpr int kRows = 128;           // rows of a slot (tensor-memory lanes)
constexpr int kTile = 128;           // positions of a tile
// Eight warps gather: the copies one warp has in flight are few (four warps reached 12 bytes a cycle and
// SM from HBM where eight reach 21).
constexpr int kGatherWarps = 8;
constexpr int kGatherRows = 2 * kTile / kGatherWarps;  // rows of a K or V tile one gather warp copies
static_assert(kGatherRows == 32, "a lane resolves one row");
constexpr int kThreads = 256 + 32 * kGatherWarps + 128;
// Registers a thread: 640 threads start with 96; the softmax warps take what the gather gives up.
constexpr int kStartRegisters = 96, kSoftmaxRegisters = 144, kGatherRegisters = 48, kOtherRegisters = 96;
static_assert(256 * kSoftmaxRegisters + 32 * kGatherWarps * kGatherRegisters + 128 * kOtherRegisters <=
                  kThreads * kStartRegisters, "more registers than the block starts with");
constexpr int kMaxEntries = EKV_ATTENTION_MAX_ROW_TILES;
// What an item costs, in a common unit: a start (queries, first keys, writing the result) and
// each tile; kBoth items of more than 128 rows, others below.  A share of equal cost per block.
constexpr int kBothStart = 24, kBothTile = 6;
constexpr int kSmallStart = 3, kSmallTile = 4;
constexpr int kPairTiles = 4;        // tiles from which a small item uses both slots
constexpr int kFewRows = 16;         // rows up to which rows_kernel takes a request
constexpr int kFewTile = 64;         // its unit of work, positions
constexpr int kFewStart = 2, kFewUnit = 1;
constexpr int kFewWarps = 8;
constexpr int kFewPrefix = 4096;     // longest prefix it takes: a part of it to a worker, joined one by one
constexpr int kLargeTime = 37, kFewTime = 35, kLeastShare = 24;
enum Mode { kSingle = 0, kBoth = 1, kPair = 2 };
constexpr int kMaskRing = 16;
constexpr int kItemRing = 8, kItemsAhead = 5;
constexpr float kRaise = 8.f;
// A row's maximum is a product of score and scale rounded to 32 bits, its weights are taken of the exact one.  Below
// kLarge the two differ by 2^-5 at most; from there on, where they come to differ by more than an exponent holds, the
// scores are rounded in the same way first.
constexpr float kLarge = 1048576.f;

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
    int64_t slots, table_rows, table_width, table_stride;
    int64_t tokens, batch, source_row;
    uint32_t page_size;
    int shared;
    int page_log2;  // -1: not a power of two
    int kv_heads, group;
    int table_es, rows_es, len_es, starts_es;
    float scale_log2;  // scale * log2(e)
    // Derived: rows per KV head, prefix row tiles, prefix tiles.
    int head_rows, prefix_row_tiles, prefix_tiles;
    int blocks;
    // Workspace.
    float* prefix_out;   // [kv_heads][head_rows][dim]: an item's first part
    float2* prefix_stat; // (maximum, sum)
    float* own_out;
    float2* own_stat;
    float* next_out;     // [blocks][256][dim]: the part a block continues
    float2* next_stat;
    uint32_t* item_span;   // of each item the first block with a tile of it, and the last << 16
    uint32_t* first_entry; // [batch]: each request's first entry
    int few_prefix, few_own, large;  // what rows_kernel does (the prefix; requests), whether attention_kernel runs
    int few_rows, workers;     // most rows of an item of rows_kernel
    float* few_out;      // [workers][few_rows][dim]: the part a worker continues
    float2* few_stat;
    uint32_t* few_span;  // as item_span, of rows_kernel's items and workers
    int* few_next;       // [workers]
    int* next_item;      // [blocks]: the item of the part a block continues, or -1
    uint32_t* failed;    // [blocks]: a wait ran out
};

// ---------------------------------------------------------------- requests

struct Request {
    int64_t begin;  // first query token
    int64_t fresh;  // query tokens
    int32_t length;
};

__device__ __forceinline__ Request request_at(const AttentionParams& p, int64_t b) {
    Request r;
    r.begin = b;
    r.fresh = 1;
    if (p.starts) {
        r.begin = load_index(p.starts, p.starts_es, b);
        r.fresh = load_index(p.starts, p.starts_es, b + 1) - r.begin;
        if (r.begin < 0 || r.fresh < 0 || r.fresh > p.tokens - r.begin) r.fresh = 0;
    }
    const int64_t length = load_index(p.lengths, p.len_es, b);
    r.length = static_cast<int32_t>(length < 0 ? 0 : (length > INT32_MAX ? INT32_MAX : length));
    return r;
}

// Request of query token n and its place in it; false for a token of no request.
__device__ __forceinline__ bool request_of(const AttentionParams& p, int64_t n, int64_t& b, Request& r) {
    if (n >= p.tokens) return false;
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
        b = low;
    }
    r = request_at(p, b);
    return n >= r.begin && n < r.begin + r.fresh;
}

// Where position j of table row `row` is looked up: the page is loaded at once and used later.
struct Lookup {
    int page;         // -1: none
    uint32_t offset;  // in the page
};

__device__ __forceinline__ Lookup look_up(const AttentionParams& p, int row, uint32_t j) {
    Lookup found{-1, 0};
    const uint32_t index = p.page_log2 >= 0 ? j >> p.page_log2 : j / p.page_size;
    if (row >= 0 && index < p.table_width) {
        const int64_t at = row * p.table_stride + index;
        if (p.table_es == 8) {
            const int64_t page = static_cast<const int64_t*>(p.tables)[at];
            found.page = page >= 0 && page < p.slots ? static_cast<int>(page) : -1;
        } else {
            found.page = static_cast<const int32_t*>(p.tables)[at];
        }
        found.offset = j - index * p.page_size;
    }
    return found;
}

// The slot, or -1 where there is none inside the planes.
__device__ __forceinline__ int slot_of(const AttentionParams& p, const Lookup& found) {
    if (found.page < 0 || found.page >= p.slots) return -1;
    const int64_t slot = static_cast<int64_t>(found.page) * p.page_size + found.offset;
    return slot < p.slots ? static_cast<int>(slot) : -1;
}

// ---------------------------------------------------------------- the list of items

// One entry per row tile of a request's own part, in shared memory; the items of an entry are
// its KV heads.
struct Plan {
    uint32_t cost[kMaxEntries + 1];  // running cost of one head
    int32_t end[kMaxEntries];        // positions the tile's last row sees
    uint16_t request[kMaxEntries];
    uint16_t row_tile[kMaxEntries];
    bool small[kMaxEntries];         // up to 128 rows
    bool few[kMaxEntries];           // up to 16: not attention_kernel's
    int64_t scratch[kThreads / 32];
    uint32_t entries;
    int blocks;  // of the grid that have work, the first ones
};

struct Cost {
    int start, tile;
};
__host__ __device__ __forceinline__ Cost cost_of(int64_t rows) {
    return rows > kRows ? Cost{kBothStart, kBothTile} : Cost{kSmallStart, kSmallTile};
}
__device__ __forceinline__ uint32_t item_cost(Cost c, int64_t tiles) {
    return tiles > 0 ? static_cast<uint32_t>(c.start + c.tile * tiles) : 0u;
}
__device__ __forceinline__ int item_tiles(Cost c, uint32_t cost) {
    return cost ? static_cast<int>((cost - c.start) / c.tile) : 0;
}

// What rows_kernel takes of a request, and its cost of one head.
__device__ __forceinline__ uint32_t few_cost(const AttentionParams& p, const Request& r) {
    const int64_t reach = p.table_width * p.page_size, end = r.length < reach ? r.length : reach;
    if (!p.few_own || r.fresh <= 0 || r.fresh * p.group > kFewRows || end <= p.shared) return 0;
    return item_cost(Cost{kFewStart, kFewUnit}, (end - p.shared + kFewTile - 1) / kFewTile);
}
__device__ __forceinline__ uint32_t few_prefix_cost(const AttentionParams& p) {
    return p.few_prefix ? item_cost(Cost{kFewStart, kFewUnit}, (p.shared + kFewTile - 1) / kFewTile) : 0;
}

// Blocks (an SM each) that attention_kernel uses when both kernels have work: the two share the SMs in
// proportion to their estimated times there (a unit of its cost takes about 0.37 us of an SM, one of
// rows_kernel's 0.35 us, at heads of 128; heads of 64 go by the same numbers), so that the memory-bound part runs beside
// the compute-bound one: 128 requests over 16384 shared tokens 181 us against 217 one behind the other where the two
// were compared, 173 now.
__device__ __forceinline__ int large_blocks(const AttentionParams& p, int64_t large, int64_t few) {
    if (!few || !large) return p.blocks;
    const int64_t mine = large * kLargeTime, its = few * kFewTime;
    int64_t blocks = (mine * p.blocks + mine + its - 1) / (mine + its);
    const int64_t most = (large + kLeastShare - 1) / kLeastShare;  // a few tiles a block at least
    if (blocks > most) blocks = most;
    if (blocks > p.blocks - 1) blocks = p.blocks - 1;
    return blocks < 1 ? 1 : static_cast<int>(blocks);
}

// Index (in the request) of the last token of a row tile.
__device__ __forceinline__ int64_t last_token(int64_t row_tile, int64_t fresh, int group) {
    const int64_t last = (row_tile * 2 * kRows + 2 * kRows - 1) / group;
    return last < fresh ? last : fresh - 1;
}

// Exclusive scan over the block; `total` is the sum of all.
__device__ __forceinline__ int64_t block_scan(int64_t value, int64_t& total, int64_t* scratch) {
    const unsigned lane = lane_id(), warp = threadIdx.x >> 5;
    int64_t sum = value;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w == warp) before = total;
        total += scratch[w];
    }
    __syncthreads();
    return before + sum - value;
}

__device__ __forceinline__ void build_plan(const AttentionParams& p, Plan& plan) {
    int64_t entries = 0, few = few_prefix_cost(p);
    for (int64_t first = 0; first < p.batch; first += kThreads) {
        const int64_t b = first + threadIdx.x;
        Request r{0, 0, 0};
        if (b < p.batch) r = request_at(p, b);
        const int64_t tiles = (r.fresh * p.group + 2 * kRows - 1) / (2 * kRows);
        int64_t total;
        const int64_t at = entries + block_scan(tiles, total, plan.scratch);
        int64_t its;
        block_scan(b < p.batch ? few_cost(p, r) : 0, its, plan.scratch);
        few += its;
        if (b < p.batch) {
            if (blockIdx.x == 0) p.first_entry[b] = static_cast<uint32_t>(at < kMaxEntries ? at : kMaxEntries);
            for (int64_t t = 0; t < tiles && at + t < kMaxEntries; ++t) {
                const int64_t seen = r.length - r.fresh + last_token(t, r.fresh, p.group) + 1;
                plan.request[at + t] = static_cast<uint16_t>(b);
                plan.row_tile[at + t] = static_cast<uint16_t>(t);
                plan.end[at + t] = static_cast<int32_t>(seen);
                plan.small[at + t] = r.fresh * p.group - t * 2 * kRows <= kRows;
                plan.few[at + t] = r.fresh * p.group <= kFewRows;
            }
        }
        entries += total;
    }
    if (entries > kMaxEntries) entries = kMaxEntries;  // only for query_starts that are not ascending
    __syncthreads();
    const int64_t reach = p.table_width * p.page_size;
    uint32_t running = 0;
    for (int64_t first = 0; first < entries; first += kThreads) {
        const int64_t e = first + threadIdx.x;
        uint32_t cost = 0;
        if (e < entries) {
            const int64_t end = plan.end[e] < reach ? plan.end[e] : reach;
            cost = item_cost(cost_of(plan.small[e] ? 1 : 2 * kRows), (end - p.shared + kTile - 1) / kTile);
            // rows_kernel takes requests of few rows.
            if (end <= p.shared || plan.few[e]) cost = 0;
        }
        int64_t total;
        const uint32_t at = running + static_cast<uint32_t>(block_scan(cost, total, plan.scratch));
        if (e < entries) plan.cost[e] = at;
        running += static_cast<uint32_t>(total);
    }
    if (threadIdx.x == 0) {
        plan.cost[entries] = running;
        plan.entries = static_cast<uint32_t>(entries);
        const int64_t prefix = p.prefix_tiles ? static_cast<int64_t>(item_cost(cost_of(p.head_rows), p.prefix_tiles)) *
                                                    p.prefix_row_tiles * p.kv_heads : 0;
        plan.blocks = large_blocks(p, prefix + static_cast<int64_t>(running) * p.kv_heads, few * p.kv_heads);
    }
    __syncthreads();
}

// Block `block`'s share of [0, total) begins here.
__device__ __forceinline__ int64_t share_begin(int64_t block, int64_t total, int blocks) {
    const int64_t product = total * block;  // below 2^63: the total is below 2^49
    if (product <= UINT32_MAX) return static_cast<uint32_t>(product) / static_cast<uint32_t>(blocks);
    return product / blocks;
}

// The block whose share holds `at`.
__device__ __forceinline__ int owner(int64_t at, int64_t total, int blocks) {
    const int64_t product = (at + 1) * blocks - 1;
    if (product <= UINT32_MAX && total <= UINT32_MAX) {
        return static_cast<int>(static_cast<uint32_t>(product) / static_cast<uint32_t>(total));
    }
    return static_cast<int>(product / total);
}

// First tile at or behind position x of an item that begins at `start` (its tile t > 0 lies at
// start + c.start + t * c.tile).
__device__ __forceinline__ int first_tile(Cost c, int64_t x, int64_t start, int tiles) {
    if (x <= start) return 0;
    const int64_t behind = x - start - c.start + c.tile - 1;
    int64_t t = behind >= 0 && behind <= UINT32_MAX ? static_cast<uint32_t>(behind) / static_cast<uint32_t>(c.tile)
                                                    : behind / c.tile;
    if (t < 1) t = 1;
    return t < tiles ? static_cast<int>(t) : tiles;
}

// The blocks that each item spans, for combine_kernel; every block of the grid writes some.
__device__ __forceinline__ void write_spans(const AttentionParams& p, const Plan& plan) {
    const Cost prefix = cost_of(p.head_rows);
    const uint32_t prefix_cost = item_cost(prefix, p.prefix_tiles);
    const int prefix_items = p.prefix_tiles ? p.prefix_row_tiles * p.kv_heads : 0;
    const int64_t prefix_total = static_cast<int64_t>(prefix_cost) * prefix_items;
    const int64_t total = prefix_total + static_cast<int64_t>(plan.cost[plan.entries]) * p.kv_heads;
    const int items = prefix_items + static_cast<int>(plan.entries) * p.kv_heads;
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < items; i += plan.blocks * kThreads) {
        Cost c = prefix;
        uint32_t cost = prefix_cost;
        int64_t start = static_cast<int64_t>(i) * prefix_cost;
        if (i >= prefix_items) {
            const int e = (i - prefix_items) / p.kv_heads, head = i - prefix_items - e * p.kv_heads;
            c = cost_of(plan.small[e] ? 1 : 2 * kRows);
            cost = plan.cost[e + 1] - plan.cost[e];
            start = prefix_total + static_cast<int64_t>(plan.cost[e]) * p.kv_heads + static_cast<int64_t>(head) * cost;
        }
        uint32_t span = 1;  // first 1, last 0: nothing
        if (cost) {
            const int tiles = item_tiles(c, cost);
            const int64_t last = start + (tiles > 1 ? c.start + static_cast<int64_t>(tiles - 1) * c.tile : 0);
            span = static_cast<uint32_t>(owner(start, total, plan.blocks)) |
                   static_cast<uint32_t>(owner(last, total, plan.blocks)) << 16;
        }
        p.item_span[i] = span;
    }
}

// Last of `count` entries whose running cost is at most x.
__device__ __forceinline__ uint32_t entry_at(const uint32_t* cost, uint32_t count, int64_t x) {
    uint32_t low = 0, high = count;
    while (high - low > 1) {
        const uint32_t mid = (low + high) >> 1;
        if (cost[mid] <= x) {
            low = mid;
        } else {
            high = mid;
        }
    }
    return low;
}

struct __align__(16) Item {
    int mode;       // Mode: how the slots share it
    int prefix;
    int first;      // this block has the item's first tile
    int head;
    int rows;       // rows of the item, up to 256; 0 ends the list
    int row;        // first row: of the head (prefix) or of the request (own)
    int low, high;  // tiles of this block
    int begin, end; // positions of the whole item
    int table_row;  // -1: no row of the table
    int id;         // prefix items first, then the own ones, entry by entry
    int token;      // query token of row 0 of the head or request
    int bias;       // own items: token i of the request sees bias + i positions
};

struct Walk {
    int64_t start, stop;  // this block's share
    int prefix_cost, prefix_items;
    int index;            // next prefix item
    uint32_t entry;
    int head;
};

__device__ __forceinline__ Walk begin_walk(const AttentionParams& p, const Plan& plan) {
    Walk w;
    w.prefix_cost = item_cost(cost_of(p.head_rows), p.prefix_tiles);
    w.prefix_items = p.prefix_tiles ? p.prefix_row_tiles * p.kv_heads : 0;
    const int64_t prefix_total = static_cast<int64_t>(w.prefix_cost) * w.prefix_items;
    const int64_t total = prefix_total + static_cast<int64_t>(plan.cost[plan.entries]) * p.kv_heads;
    w.start = share_begin(blockIdx.x, total, plan.blocks);
    w.stop = share_begin(blockIdx.x + 1, total, plan.blocks);
    w.index = w.prefix_items;
    w.entry = 0;
    w.head = 0;
    if (w.start < prefix_total) {
        w.index = static_cast<int>(w.start / w.prefix_cost);
    } else if (plan.entries) {
        const int64_t x = w.start - prefix_total;
        w.entry = entry_at(plan.cost, plan.entries, x / p.kv_heads);
        const int64_t cost = plan.cost[w.entry + 1] - plan.cost[w.entry];
        if (cost) w.head = static_cast<int>((x - static_cast<int64_t>(plan.cost[w.entry]) * p.kv_heads) / cost);
    }
    return w;
}

// The next item of which this block has a tile; false at the end of its share.
__device__ __forceinline__ bool next_item(const AttentionParams& p, const Plan& plan, Walk& w, Item& item) {
    while (w.index < w.prefix_items) {
        const int64_t start = static_cast<int64_t>(w.index) * w.prefix_cost;
        if (start >= w.stop) return false;
        const int i = w.index++;
        const Cost c = cost_of(p.head_rows);
        item.low = first_tile(c, w.start, start, p.prefix_tiles);
        item.high = first_tile(c, w.stop, start, p.prefix_tiles);
        if (item.low >= item.high) continue;
        item.prefix = 1;
        item.id = i;
        item.first = item.low == 0;
        item.head = i / p.prefix_row_tiles;
        item.row = (i - item.head * p.prefix_row_tiles) * 2 * kRows;
        item.rows = p.head_rows - item.row < 2 * kRows ? p.head_rows - item.row : 2 * kRows;
        item.table_row = static_cast<int>(p.source_row);
        item.token = 0;
        item.bias = 0;
        item.begin = 0;
        item.end = p.shared;
        return true;
    }
    const int64_t prefix_total = static_cast<int64_t>(w.prefix_cost) * w.prefix_items;
    while (w.entry < plan.entries) {
        const int64_t cost = plan.cost[w.entry + 1] - plan.cost[w.entry];
        const int64_t start = prefix_total + static_cast<int64_t>(plan.cost[w.entry]) * p.kv_heads + w.head * cost;
        if (cost && start >= w.stop) return false;
        const uint32_t e = w.entry;
        const int head = w.head;
        if (!cost || ++w.head >= p.kv_heads) {
            // The next entry that costs anything.
            const uint32_t done = plan.cost[w.entry + 1];
            const uint32_t found = entry_at(plan.cost, plan.entries, done);
            w.entry = found > w.entry && done < plan.cost[plan.entries] ? found : plan.entries;
            w.head = 0;
        }
        if (!cost) continue;
        const Cost c = cost_of(plan.small[e] ? 1 : 2 * kRows);
        const int tiles = item_tiles(c, static_cast<uint32_t>(cost));
        item.low = first_tile(c, w.start, start, tiles);
        item.high = first_tile(c, w.stop, start, tiles);
        if (item.low >= item.high) continue;
        const int64_t reach = p.table_width * p.page_size;
        item.prefix = 0;
        item.id = w.prefix_items + static_cast<int>(e) * p.kv_heads + head;
        item.first = item.low == 0;
        item.head = head;
        const int64_t b = plan.request[e];
        const Request request = request_at(p, b);
        item.row = plan.row_tile[e] * 2 * kRows;
        const int left = static_cast<int>(request.fresh) * p.group - item.row;
        item.rows = left < 2 * kRows ? left : 2 * kRows;
        const int64_t table_row = p.rows ? load_index(p.rows, p.rows_es, b) : b;
        item.table_row = table_row >= 0 && table_row < p.table_rows ? static_cast<int>(table_row) : -1;
        item.token = static_cast<int>(request.begin);
        item.bias = static_cast<int>(request.length - request.fresh + 1);
        item.begin = p.shared;
        item.end = plan.end[e] < reach ? plan.end[e] : static_cast<int>(reach);
        return true;
    }
    return false;
}

__device__ __forceinline__ int mode_of(const Item& item) {
    return item.rows > kRows ? kBoth : (item.high - item.low >= kPairTiles ? kPair : kSingle);
}

// Positions that an item's row sees; false for a row of no request.
__device__ __forceinline__ bool row_sees(const AttentionParams& p, const Item& item, int r, int64_t& seen) {
    if (r >= item.rows) return false;
    const int at = (item.row + r) / p.group;
    seen = item.bias + at;
    if (!item.prefix) return true;
    int64_t b;
    Request request;
    if (!request_of(p, at, b, request)) return false;
    seen = request.length - request.fresh + (at - request.begin) + 1;
    return true;
}

// ---------------------------------------------------------------- the kernel

template <int kDim>
struct Layout {
    static constexpr int kStages = kDim == 128 ? 2 : 4;
    static constexpr uint32_t kBlock = kTile * 128;            // 128 rows of 128 bytes
    static constexpr uint32_t kOperand = kBlock * (kDim / 64); // 128 rows of the head dimension
    static constexpr uint32_t kQuery = 0;
    static constexpr uint32_t kKeys = 2 * kOperand;
    static constexpr uint32_t kValues = kKeys + kStages * kOperand;
    static constexpr uint32_t kPlan = kValues + kStages * kOperand;
    static constexpr uint32_t kItems = kPlan + ((sizeof(Plan) + 15) / 16) * 16;
    static constexpr uint32_t kMasks = kItems + kItemRing * sizeof(Item);
    static constexpr uint32_t kStats = kMasks + kMaskRing * 16;  // maximum and sum of each row, of both slots
    static constexpr uint32_t kBarriers = kStats + 2 * kRows * 8;
    // Six of each stage, nine of each slot, two of each place in the item ring, one where the slots of a pair meet.
    static constexpr int kBarrierCount = 6 * kStages + 9 * 2 + 2 * kItemRing + 1;
    static constexpr uint32_t kTail = kBarriers + kBarrierCount * 8;
    static constexpr uint32_t kBytes = kTail + 16;  // tensor-memory address, failed flag, V tiles passed on
};

template <typename T>
struct Kind;
template <>
struct Kind<__nv_bfloat16> {
    static constexpr bool kBf16 = true;
    static constexpr float kShift = 0.f, kFactor = 1.f;  // of the weights: 2^kShift
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
    }
};
template <>
struct Kind<__half> {
    static constexpr bool kBf16 = false;
    static constexpr float kShift = 7.f, kFactor = 128.f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    }
};

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(const __grid_constant__ AttentionParams p) {
    using L = Layout<kDim>;
    extern __shared__ __align__(1024) uint8_t shared[];
    Plan& plan = *reinterpret_cast<Plan*>(shared + L::kPlan);
    uint4* masks = reinterpret_cast<uint4*>(shared + L::kMasks);
    volatile uint32_t* failed = reinterpret_cast<uint32_t*>(shared + L::kTail + 4);
    const uint32_t base = shared_address(shared);
    constexpr int kIssueWarp = 8 + kGatherWarps;
    const int warp = threadIdx.x >> 5;
    const unsigned lane = lane_id();

    // K and V stages: landed (written), full (and visible to the tensor cores), empty (read).
    const uint32_t barriers = base + L::kBarriers;
    const auto stage_barrier = [&](int which, int s) { return barriers + 8 * (which * L::kStages + s); };
    const auto k_landed = [&](int s) { return stage_barrier(0, s); };
    const auto k_full = [&](int s) { return stage_barrier(1, s); };
    const auto k_empty = [&](int s) { return stage_barrier(2, s); };
    const auto v_landed = [&](int s) { return stage_barrier(3, s); };
    const auto v_full = [&](int s) { return stage_barrier(4, s); };
    const auto v_empty = [&](int s) { return stage_barrier(5, s); };
    const auto slot_barrier = [&](int which, int s) { return barriers + 8 * (6 * L::kStages + 2 * which + s); };
    const auto q_landed = [&](int s) { return slot_barrier(0, s); };
    const auto q_full = [&](int s) { return slot_barrier(1, s); };
    const auto s_full = [&](int s, int half) { return slot_barrier(2 + half, s); };  // scores of half a tile
    const auto p_full = [&](int s, int half) { return slot_barrier(4 + half, s); };  // its weights
    const auto o_half = [&](int s) { return slot_barrier(6, s); };                   // added to the output
    const auto o_full = [&](int s) { return slot_barrier(7, s); };                   // the item's last one too
    const auto drain = [&](int s) { return slot_barrier(8, s); };
    const auto item_full = [&](int i) { return barriers + 8 * (6 * L::kStages + 18 + i); };
    const auto item_empty = [&](int i) { return barriers + 8 * (6 * L::kStages + 18 + kItemRing + i); };
    const uint32_t v_count = base + L::kTail + 8;  // V tiles that are passed on
    const uint32_t meet = barriers + 8 * (L::kBarrierCount - 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            barrier_init(k_landed(s), 16 * kGatherWarps);
            barrier_init(k_full(s), 1);
            barrier_init(k_empty(s), 2);  // both slots, or one of them and the warp that passes on
            barrier_init(v_landed(s), 16 * kGatherWarps);
            barrier_init(v_full(s), 1);
            barrier_init(v_empty(s), 2);
        }
        for (int s = 0; s < 2; ++s) {
            barrier_init(q_landed(s), kRows);
            barrier_init(q_full(s), 1);
            for (int half = 0; half < 2; ++half) {
                barrier_init(s_full(s, half), 1);
                barrier_init(p_full(s, half), 4);
            }
            barrier_init(o_half(s), 1);
            barrier_init(o_full(s), 1);
            barrier_init(drain(s), 1);
        }
        barrier_init(meet, 8);
        for (int i = 0; i < kItemRing; ++i) {
            barrier_init(item_full(i), 1);
            barrier_init(item_empty(i), 8 + kGatherWarps + 3);  // every warp but the one that walks
        }
        *failed = 0;
        count_store(v_count, 0);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    grid_dependency_wait();
    allow_dependents();  // rows_kernel needs nothing of this one: its blocks begin where this one's leave room
    // Behind the wait: a block of the kernel before may still need tensor memory on this SM.
    if (warp == kIssueWarp) tensor_alloc(base + L::kTail, 512);
    tensor_fence_before();
    build_plan(p, plan);  // ends with __syncthreads
    tensor_fence_after();
    const uint32_t tensor = *reinterpret_cast<volatile uint32_t*>(shared + L::kTail);
    if (static_cast<int>(blockIdx.x) >= plan.blocks) {  // rows_kernel's SM
        if (warp == kIssueWarp) tensor_free(tensor, 512);
        return;
    }
    write_spans(p, plan);

    // A row of an operand is copied 16 bytes a lane, kAtOnce rows a step; its chunks are
    // swizzled within their 128 bytes by the row's place in its eight.
    constexpr int kLanes = kDim / 8, kAtOnce = 32 / kLanes;
    const int chunk = lane % kLanes, sub = lane / kLanes;
    const auto target = [&](uint32_t operand, int row) {
        return operand + (chunk >> 3) * L::kBlock + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
    };
    Item* items = reinterpret_cast<Item*>(shared + L::kItems);
    Item item;
    uint32_t item_uses = 0;
    int turn = 0;  // slot of the next item of up to 128 rows
    // The next item, for a whole warp or one thread of it; false at the list's end (or a failed wait).
    const auto next = [&](bool alone) {
        const int place = item_uses % kItemRing;
        bool there = barrier_wait(item_full(place), (item_uses / kItemRing) & 1, failed);
        if (!alone) there = __all_sync(0xffffffffu, there);
        if (!there) return false;
        item = items[place];
        if (!alone) __syncwarp();
        if (alone || lane == 0) barrier_arrive(item_empty(place));
        ++item_uses;
        return item.rows > 0;
    };

    if (warp < 8) {
        // ------------------------------------------------------------ softmax of slot `slot`
        registers_grow<kSoftmaxRegisters>();
        const int slot = warp >> 2;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 tensor-memory lanes a warp
        const uint32_t scores = tensor + lanes + slot * kTile;
        const uint32_t output = tensor + lanes + 256 + slot * 128;
        uint32_t uses = 0, halves = 0, ends = 0, tiles_before = 0, meetings = 0;
        const int r = (warp & 3) * 32 + lane;
        float2* stats = reinterpret_cast<float2*>(shared + L::kStats);
        // The items this slot has a part in, one ahead: its queries are copied (each warp its 32 rows)
        // once the products with the ones before are complete.  An item stays in the ring until it is done.
        int ahead = -1;        // its place in the ring; -1: none
        uint32_t ahead_tiles = 0;  // tiles of the block before it
        const auto release = [&](int place) {
            __syncwarp();
            if (lane == 0) barrier_arrive(item_empty(place));
        };
        const auto prepare = [&]() {
            ahead = -1;
            while (true) {
                const int place = item_uses % kItemRing;
                if (!__all_sync(0xffffffffu, barrier_wait(item_full(place), (item_uses / kItemRing) & 1, failed))) return false;
                ++item_uses;
                const Item& its = items[place];
                const int rows = its.rows, mode = its.mode;
                if (!rows) return true;
                ahead_tiles = tiles_before;
                tiles_before += static_cast<uint32_t>(its.high - its.low);
                if (mode == kSingle) {
                    const int owner_slot = turn;
                    turn ^= 1;
                    if (owner_slot != slot) {
                        release(place);
                        continue;
                    }
                }
                ahead = place;
                const int first = (mode == kBoth ? slot * kRows : 0) + (warp & 3) * 32;
                const int row = its.row, head = its.head * p.group, token = its.token;
                const uint32_t operand = base + L::kQuery + slot * L::kOperand;
#pragma unroll 1
                for (int i = sub; i < 32 && first + i - sub < rows; i += kAtOnce) {
                    if (first + i >= rows) break;
                    const int local = row + first + i;
                    const int at = local / p.group;
                    copy16_async(target(operand, (warp & 3) * 32 + i),
                                 static_cast<const char*>(p.query) + 16 * chunk +
                                     2 * ((token + at) * p.q_token + (head + local - at * p.group) * p.q_head), 16);
                }
                copies_arrive(q_landed(slot));
                return true;
            }
        };
        if (!prepare()) goto finish;
        while (ahead >= 0) {
            const int place = ahead;
            const uint32_t tiles = ahead_tiles;
            const Item& item = items[place];
            const bool both = item.mode == kBoth, pair = item.mode == kPair;
            const int item_row = (both ? slot * kRows : 0) + r;
            int64_t seen;
            const bool present = row_sees(p, item, item_row, seen);
            // Positions from the item's first one on; a row of no request is computed with the others and dropped.
            const int64_t reach = seen - item.begin;
            const int limit = !present || reach > INT32_MAX ? INT32_MAX : (reach < 0 ? 0 : static_cast<int>(reach));
            const bool idle = (both ? slot * kRows : 0) + (warp & 3) * 32 >= item.rows;  // no row in this warp
            float top = -INFINITY;
            float2 total = make_float2(0.f, 0.f);
            const int low = item.low + (pair ? slot : 0), high = item.high, step = pair ? 2 : 1;
            const uint32_t mask_base = tiles - item.low;
            for (int t = low; t < high; t += step, ++uses) {
#pragma unroll 1
                for (int half = 0; half < 2; ++half, ++halves) {
                    if (!__all_sync(0xffffffffu, barrier_wait(s_full(slot, half), uses & 1, failed))) goto finish;
                    tensor_fence_after();
                    if (half && t + step >= high && !prepare()) goto finish;
                    if (!idle) {
                        const uint32_t mine = scores + 64 * half;
                        uint32_t s[64];
                        tensor_load32(mine, s);
                        tensor_load32(mine + 32, s + 32);
                        // Positions this row sees here: those that have a slot, up to its last.
                        const int left = limit - t * kTile - 64 * half;
                        const uint2 there = reinterpret_cast<const uint2*>(&masks[(mask_base + t) % kMaskRing])[half];
                        const bool whole = __all_sync(0xffffffffu, left >= 64) && (there.x & there.y) == 0xffffffffu;
                        tensor_wait_load();
                        if (!whole) {
                            const auto until = [](int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); };
                            const uint32_t first = there.x & until(left), second = there.y & until(left - 32);
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                if (!(first >> j & 1u)) s[j] = 0xff800000u;  // -inf
                                if (!(second >> j & 1u)) s[32 + j] = 0xff800000u;
                            }
                        }
                        float highs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int j = 0; j < 64; j += 8) {
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                highs[c] = max3(highs[c], __uint_as_float(s[j + 2 * c]), __uint_as_float(s[j + 2 * c + 1]));
                            }
                        }
                        const float most = fmaxf(fmaxf(highs[0], highs[1]), fmaxf(highs[2], highs[3])) * p.scale_log2;
                        const bool raise = present && most - top > kRaise;  // exact where it matters, as top + kRaise is not
                        if (__any_sync(0xffffffffu, raise)) {
                            const float before = top;
                            if (raise) top = most;
                            const float factor = raise ? (before == -INFINITY ? 0.f : exp2_approx(before - top)) : 1.f;
                            total.x *= factor;
                            total.y *= factor;
                            if (t > low || half) {
                                // The weights so far are all in the output before it is scaled (those before the last
                                // half's are: the product behind them gave these scores).
                                if (!__all_sync(0xffffffffu, barrier_wait(o_half(slot), (halves - 1) & 1, failed))) goto finish;
                                tensor_fence_after();
#pragma unroll 1
                                for (int c = 0; c < kDim / 16; ++c) {
                                    uint32_t o[16];
                                    tensor_load16(output + 16 * c, o);
                                    tensor_wait_load();
#pragma unroll
                                    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * factor);
                                    tensor_store16(output + 16 * c, o);
                                }
                            }
                        }
                        float shift = top == -INFINITY ? 0.f : Kind<T>::kShift - top, scale = p.scale_log2;
                        if (__any_sync(0xffffffffu, fabsf(shift) >= kLarge)) {
                            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                            for (int j = 0; j < 64; ++j) {
                                s[j] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(s[j]), scale), base));
                            }
                            scale = 1.f;
                            shift = Kind<T>::kShift;
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint32_t weights[16];
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                const int at = 32 * c + j;
                                float2 x = fma2(make_float2(__uint_as_float(s[at]), __uint_as_float(s[at + 1])),
                                                make_float2(scale, scale), make_float2(shift, shift));
                                x.x = exp2_approx(x.x);
                                x.y = exp2_approx(x.y);
                                total = add2(total, x);
                                weights[j / 2] = Kind<T>::pack(x.x, x.y);
                            }
                            tensor_store16(mine + 16 * c, weights);
                        }
                        tensor_wait_store();
                    }
                    tensor_fence_before();
                    __syncwarp();
                    if (lane == 0) barrier_arrive(p_full(slot, half));
                }
            }
            if (!__all_sync(0xffffffffu, barrier_wait(o_full(slot), ends & 1, failed))) goto finish;
            ++ends;
            tensor_fence_after();
            float sum = total.x + total.y, factor = 1.f, other = 0.f;
            if (pair) {
                // The slots exchange their maxima and sums; each then joins half of the columns, reading the other
                // slot's too: what that one's products and rescaling have written lies before the meeting.
                stats[slot * kRows + r] = make_float2(top, sum);
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(meet);
                if (!__all_sync(0xffffffffu, barrier_wait(meet, meetings & 1, failed))) goto finish;
                tensor_fence_after();
                ++meetings;
                const float2 its = stats[(slot ^ 1) * kRows + r];
                const float higher = fmaxf(top, its.x);
                if (higher > -INFINITY) {
                    factor = exp2_approx(top - higher);
                    other = exp2_approx(its.x - higher);
                }
                top = higher;
                sum = sum * factor + its.y * other;
            }
            if (!idle) {
                float* partial;
                float2* stat;
                if (item.first) {
                    // Rows of a head in token order: an own item's lie behind its request's first token.
                    const int64_t row = static_cast<int64_t>(item.head) * p.head_rows +
                                        static_cast<int64_t>(item.token) * p.group + item.row + item_row;
                    partial = (item.prefix ? p.prefix_out : p.own_out) + row * kDim;
                    stat = (item.prefix ? p.prefix_stat : p.own_stat) + row;
                } else {
                    const int64_t row = static_cast<int64_t>(blockIdx.x) * 2 * kRows + item_row;
                    partial = p.next_out + row * kDim;
                    stat = p.next_stat + row;
                }
                const int first = pair ? slot * (kDim / 2) : 0, last = pair ? first + kDim / 2 : kDim;
                const uint32_t peer = tensor + lanes + 256 + (slot ^ 1) * 128;
#pragma unroll 1
                for (int c = first; c < last; c += 32) {
                    uint32_t o[32], q[32];
                    tensor_load32(output + c, o);
                    if (pair) tensor_load32(peer + c, q);
                    tensor_wait_load();
                    if (pair) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            o[j] = __float_as_uint(__uint_as_float(o[j]) * factor + __uint_as_float(q[j]) * other);
                        }
                    }
                    if (present) {
#pragma unroll
                        for (int j = 0; j < 32; j += 8) store_sector(partial + c + j, o + j);
                    }
                }
                if (present && (!pair || slot == 0)) *stat = make_float2(top, sum);
                tensor_fence_before();
            }
            if (pair) {  // neither slot goes on before the other has read its columns
                __syncwarp();
                if (lane == 0) barrier_arrive(meet);
                if (!__all_sync(0xffffffffu, barrier_wait(meet, meetings & 1, failed))) goto finish;
                ++meetings;
                tensor_fence_after();
            }
            release(place);
        }
    } else if (warp < kIssueWarp) {
        // ------------------------------------------------------------ gather
        registers_shrink<kGatherRegisters>();
        const bool keys = warp < 8 + kGatherWarps / 2;
        const int first_row = (warp - 8) % (kGatherWarps / 2) * kGatherRows;  // of every operand
        const char* query = static_cast<const char*>(p.query) + 16 * chunk;
        const int64_t stride = 2 * (keys ? p.k_slot : p.v_slot);
        // Where this lane's copies of a stage go: the swizzle repeats every eight rows.
        constexpr int kPlaces = 8 / kAtOnce;
        uint32_t places[kPlaces];
#pragma unroll
        for (int i = 0; i < kPlaces; ++i) {
            places[i] = target(base + (keys ? L::kKeys : L::kValues), first_row + i * kAtOnce + sub);
        }
        uint32_t uses = 0;
        // This lane's row in tile t of the item.
        const auto find = [&](int t) {
            const int position = item.begin + t * kTile + first_row + static_cast<int>(lane);
            return look_up(p, position < item.end ? item.table_row : -1, static_cast<uint32_t>(position));
        };
        bool more = next(false);
        Lookup found{-1, 0};
        if (more) found = find(item.low);
        while (more) {
            const char* plane = (keys ? static_cast<const char*>(p.k_plane) + 2 * item.head * p.k_head
                                      : static_cast<const char*>(p.v_plane) + 2 * item.head * p.v_head) + 16 * chunk;
            const int high = item.high;
            for (int t = item.low; t < high; ++t, ++uses) {
                const int stage = uses % L::kStages;
                const uint32_t parity = ((uses / L::kStages) & 1) ^ 1;
                const int now = slot_of(p, found);
                // The next tile's pages are on their way while this one's rows are copied.
                if (t + 1 < high) {
                    found = find(t + 1);
                } else {
                    more = next(false);
                    if (more) found = find(item.low);
                }
                const uint32_t there = __ballot_sync(0xffffffffu, now >= 0);
                if (!__all_sync(0xffffffffu, barrier_wait(keys ? k_empty(stage) : v_empty(stage), parity, failed))) goto finish;
                // The first product of tile n - kStages is complete.  A slot's products wait for the softmax of
                // its tile before, and items that leave the other slot alone have few tiles, so
                // masks of tiles further back than kStages + kPairTiles are no longer read.
                if (keys && lane == 0) reinterpret_cast<uint32_t*>(&masks[uses % kMaskRing])[warp - 8] = there;
                const uint32_t operand = stage * L::kOperand;
                if (there == 0xffffffffu) {
#pragma unroll
                    for (int i = 0; i < kGatherRows; i += kAtOnce) {
                        const int slot = __shfl_sync(0xffffffffu, now, i + sub);
                        copy16_async(places[i / kAtOnce % kPlaces] + operand + (i / 8) * 1024, plane + slot * stride, 16);
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < kGatherRows; i += kAtOnce) {
                        const int slot = __shfl_sync(0xffffffffu, now, i + sub);
                        copy16_async(target(base + (keys ? L::kKeys : L::kValues) + operand, first_row + i + sub),
                                     slot >= 0 ? plane + slot * stride : query, slot >= 0 ? 16 : 0);
                    }
                }
                copies_arrive(keys ? k_landed(stage) : v_landed(stage));
            }
        }
    } else if (lane == 0) {
        if (warp < kIssueWarp + 2) {
            // -------------------------------------------------------- products of slot `slot`
            constexpr uint32_t kScoreProduct = mma_descriptor(Kind<T>::kBf16, kRows, kTile / 2, false);
            constexpr uint32_t kOutputProduct = mma_descriptor(Kind<T>::kBf16, kRows, kDim, true);
            const int slot = warp - kIssueWarp;
            const uint32_t scores = tensor + slot * kTile, output = tensor + 256 + slot * 128;
            const uint64_t queries = shared_operand(base + L::kQuery + slot * L::kOperand, 16);
            const uint64_t all_keys = shared_operand(base + L::kKeys, 16);
            const uint64_t all_values = shared_operand(base + L::kValues, L::kBlock);
            uint32_t uses = 0, q_uses = 0, p_uses = 0;
            bool fine = true;
            const auto parity = [&](uint32_t use) { return (use / L::kStages) & 1; };
            // A barrier tells apart only the phase under way and the one before, but a slot may come to a V tile
            // while one of the other slot's is awaited at the same stage; so it first sees that one passed on.
            // (K tiles need no such wait: an item's queries are passed on behind the K tiles of the items before.)
            const auto values_there = [&](uint32_t use) {
                return (use < L::kStages || count_wait(v_count, use - L::kStages + 1, failed)) &&
                       barrier_wait(v_full(use % L::kStages), parity(use), failed);
            };
            while (fine && next(true)) {
                const bool pair = item.mode == kPair;
                const uint32_t before = uses - item.low;  // tile t of the item is the block's tile before + t
                uses += item.high - item.low;
                if (item.mode == kSingle) {
                    const int owner = turn;
                    turn ^= 1;
                    if (owner != slot) continue;
                }
                const int low = item.low + (pair ? slot : 0), high = item.high, step = pair ? 2 : 1;
                if (!(fine = barrier_wait(q_full(slot), q_uses & 1, failed))) break;
                ++q_uses;
                // Scores of half a tile; then, as soon as the weights of a half are there, their product
                // with V, and right behind it the scores of that half of the next tile, so that
                // the softmax of one half runs beside the products of the other.
                const auto score = [&](uint32_t use, int half) {
                    const uint64_t keys = all_keys + (use % L::kStages) * (L::kOperand >> 4) + half * (64 * 128 >> 4);
#pragma unroll
                    for (int k = 0; k < kDim / 16; ++k) {
                        const uint32_t step = (k / 4) * (L::kBlock >> 4) + (k % 4) * 2;
                        mma_shared(scores + 64 * half, queries + step, keys + step, kScoreProduct, k > 0);
                    }
                    mma_commit(s_full(slot, half));
                };
                uint32_t use = before + low;
                if (!(fine = barrier_wait(k_full(use % L::kStages), parity(use), failed))) break;
                tensor_fence_after();
                score(use, 0);
                score(use, 1);
                mma_commit(k_empty(use % L::kStages));
                for (int t = low; t < high; t += step, use += step, ++p_uses) {
                    const int stage = use % L::kStages;
                    const uint32_t next_use = use + step;
                    const bool more = t + step < high;
                    if (!(fine = values_there(use))) break;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        const uint64_t values = all_values + stage * (L::kOperand >> 4) + half * (64 * 128 >> 4);
                        if (!(fine = barrier_wait(p_full(slot, half), p_uses & 1, failed))) break;
                        tensor_fence_after();
#pragma unroll
                        for (int k = 0; k < kTile / 32; ++k) {
                            mma_tensor(output, scores + 64 * half + 8 * k, values + k * (16 * 128 >> 4), kOutputProduct,
                                       t > low || half > 0 || k > 0);
                        }
                        mma_commit(o_half(slot));
                        if (half) mma_commit(v_empty(stage));
                        if (!more) continue;
                        if (!half) {
                            if (!(fine = barrier_wait(k_full(next_use % L::kStages), parity(next_use), failed))) break;
                            tensor_fence_after();
                        }
                        score(next_use, half);
                        if (half) mma_commit(k_empty(next_use % L::kStages));
                    }
                    if (!fine) break;
                }
                if (fine) mma_commit(o_full(slot));
            }
            // Nothing may still use tensor memory when it is freed, whatever happened above.
            mma_commit(drain(slot));
            volatile uint32_t ran_out = 0;
            barrier_wait(drain(slot), 0, &ran_out);
        } else {
            // -------------------------------------------------------- what the gather has written, and the items
            const bool keys = warp == kIssueWarp + 3;
            uint32_t uses = 0, q_uses[2] = {0, 0};
            const auto pass_on = [&](uint32_t landed, uint32_t full, uint32_t parity) {
                if (!barrier_wait(landed, parity, failed)) return false;
                fence_async_shared();
                barrier_arrive(full);
                return true;
            };
            const auto pass_tiles = [&](const Item& its) {
                bool fine = true;
                for (int t = its.low; fine && t < its.high; ++t, ++uses) {
                    const int stage = uses % L::kStages;
                    const uint32_t parity = (uses / L::kStages) & 1;
                    fine = keys ? pass_on(k_landed(stage), k_full(stage), parity)
                                : pass_on(v_landed(stage), v_full(stage), parity);
                    if (fine && !keys) count_store(v_count, uses + 1);
                    // For the slot that has no use for the tile.
                    if (fine && its.mode != kBoth) barrier_arrive(keys ? k_empty(stage) : v_empty(stage));
                }
                return fine;
            };
            bool fine = true;
            if (keys) {
                while (fine && next(true)) {
                    for (int use = 0; fine && use < (item.mode == kSingle ? 1 : 2); ++use) {
                        const int slot = item.mode == kSingle ? turn : use;
                        fine = pass_on(q_landed(slot), q_full(slot), q_uses[slot] & 1);
                        ++q_uses[slot];
                    }
                    if (item.mode == kSingle) turn ^= 1;
                    fine = fine && pass_tiles(item);
                }
            } else {
                Walk walk = begin_walk(p, plan);
                bool more = true;
                for (uint32_t i = 0; fine; ++i) {
                    while (fine && more && item_uses < i + kItemsAhead) {
                        more = next_item(p, plan, walk, item);
                        if (!item_uses) p.next_item[blockIdx.x] = more && !item.first ? item.id : -1;
                        if (!more) item.rows = 0;
                        item.mode = mode_of(item);
                        const int place = item_uses % kItemRing;
                        fine = barrier_wait(item_empty(place), ((item_uses / kItemRing) & 1) ^ 1, failed);
                        if (!fine) break;
                        items[place] = item;
                        barrier_arrive(item_full(place));
                        ++item_uses;
                    }
                    const Item its = items[i % kItemRing];
                    if (!its.rows) break;
                    fine = fine && pass_tiles(its);
                }
            }
        }
    }
finish:
    copies_wait_all();
    __syncthreads();
    if (threadIdx.x == 0) p.failed[blockIdx.x] = *failed;
    if (warp == kIssueWarp) {
        __syncwarp();
        tensor_free(tensor, 512);
    }
}

// ---------------------------------------------------------------- few rows

template <int kDim>
struct FewLayout {
    static constexpr int kChunk = 2048 / kDim;             // positions a warp has in shared memory
    static constexpr uint32_t kOperand = kChunk * kDim * 2;  // 4096 bytes of K, as many of V
    static constexpr uint32_t kWarp = 2 * kOperand + kFewRows * kDim * 2;
    static constexpr uint32_t kPlan = kFewWarps * kWarp;
    static constexpr uint32_t kBytes = kPlan + (kMaxEntries + 2) * 4 + (kFewWarps + 1) * 8;
};

// Requests of up to 16 query rows (a decode step), and a short prefix of a small batch: too few rows to
// fill a tensor-core tile, so HBM bounds them (the own positions of 128 requests, 0.5 GB: 92 us alone on the
// GPU, 5.6 TB/s).  Work is cut as above, into equal shares of 64-position
// units, but a share belongs to a WARP, which keeps to itself: it copies 16 or 32 positions of K and V at a
// time into its own shared memory (the next keys while it weighs these, the next values while it
// scores those) and multiplies them with mma.sync, positions by rows: S^T = K Q^T, O^T += V^T P^T,
// so that up to 8 rows cost half of what 16 do.  Sixteen such warps an SM have 128 KB of buffers, about half of
// them on the way at a time.  (At heads of 128 a thread's 128 registers spill some 160 bytes.)
template <typename T, int kDim>
__global__ void __launch_bounds__(32 * kFewWarps, 2) rows_kernel(const __grid_constant__ AttentionParams p) {
    using L = FewLayout<kDim>;
    constexpr int kChunk = L::kChunk, kBlocks = kChunk / 16;  // blocks of 16 positions in a chunk
    constexpr int kLanes = kDim / 8, kAtOnce = 32 / kLanes;
    extern __shared__ __align__(1024) uint8_t shared[];
    uint32_t* running = reinterpret_cast<uint32_t*>(shared + L::kPlan);  // running cost of one head, by group
    int64_t* scratch = reinterpret_cast<int64_t*>(shared + L::kPlan + (kMaxEntries + 2) * 4);
    const int warp = threadIdx.x >> 5, lane = static_cast<int>(lane_id());
    if (!p.large) grid_dependency_wait();  // else attention_kernel, launched before, has waited
    allow_dependents();
    // Group 0 is the prefix where rows_kernel takes it, the others are the requests.
    const int offset = p.few_prefix, groups = static_cast<int>(p.batch) + offset;
    const int64_t reach = p.table_width * p.page_size;
    const Cost cost_unit{kFewStart, kFewUnit};
    uint32_t total32 = 0;
    int64_t large = 0;  // attention_kernel's cost, of one head
    for (int first = 0; first < groups; first += 32 * kFewWarps) {
        const int i = first + static_cast<int>(threadIdx.x);
        uint32_t cost = 0;
        if (i < offset) {
            cost = few_prefix_cost(p);
        } else if (i < groups) {
            const Request r = request_at(p, i - offset);
            cost = few_cost(p, r);
            if (p.large && r.fresh * p.group > kFewRows) {
                for (int64_t t = 0; t * 2 * kRows < r.fresh * p.group; ++t) {
                    const int64_t seen = r.length - r.fresh + last_token(t, r.fresh, p.group) + 1;
                    const int64_t tiles = ((seen < reach ? seen : reach) - p.shared + kTile - 1) / kTile;
                    large += item_cost(cost_of(r.fresh * p.group - t * 2 * kRows), tiles);
                }
            }
        }
        // Exclusive scan of the costs of 256 groups.
        int64_t sum = cost;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += up;
        }
        __syncthreads();
        if (lane == 31) scratch[warp] = sum;
        __syncthreads();
        int64_t before = 0, all = 0;
        for (int w = 0; w < kFewWarps; ++w) {
            if (w == warp) before = all;
            all += scratch[w];
        }
        if (i < groups) running[i] = total32 + static_cast<uint32_t>(before + sum - cost);
        total32 += static_cast<uint32_t>(all);
    }
    if (threadIdx.x == 0) running[groups] = total32;
#pragma unroll
    for (int d = 16; d; d >>= 1) large += __shfl_xor_sync(0xffffffffu, large, d);
    __syncthreads();
    if (lane == 0) scratch[warp] = large;
    __syncthreads();
    large = 0;
    for (int w = 0; w < kFewWarps; ++w) large += scratch[w];
    if (p.prefix_tiles) large += static_cast<int64_t>(item_cost(cost_of(p.head_rows), p.prefix_tiles)) * p.prefix_row_tiles;
    const int64_t total = static_cast<int64_t>(total32) * p.kv_heads;
    // The SMs that attention_kernel leaves take two blocks each.
    int blocks = static_cast<int>(gridDim.x);
    if (p.large && large && total) blocks = 2 * (p.blocks - large_blocks(p, large * p.kv_heads, total));
    if (static_cast<int>(blockIdx.x) >= blocks) return;
    // Little work goes to as many warps as it has units, an SM after another, so that its parts lie close together.
    const int workers = total < blocks * kFewWarps ? (total ? static_cast<int>(total) : 1) : blocks * kFewWarps;
    // What combine_kernel reads of the items.
    for (int i = blockIdx.x * 32 * kFewWarps + threadIdx.x; i < groups * p.kv_heads; i += blocks * 32 * kFewWarps) {
        const int group = i / p.kv_heads, head = i - group * p.kv_heads;
        const uint32_t cost = running[group + 1] - running[group];
        uint32_t span = 1;
        if (cost) {
            const int64_t start = static_cast<int64_t>(running[group]) * p.kv_heads + static_cast<int64_t>(head) * cost;
            const int units = item_tiles(cost_unit, cost);
            const int64_t last = start + (units > 1 ? kFewStart + static_cast<int64_t>(units - 1) * kFewUnit : 0);
            span = static_cast<uint32_t>(owner(start, total, workers)) |
                   static_cast<uint32_t>(owner(last, total, workers)) << 16;
        }
        p.few_span[i] = span;
    }
    const int worker = warp * blocks + blockIdx.x;
    const int64_t share = worker < workers ? share_begin(worker, total, workers) : 0;
    const int64_t stop = worker < workers ? share_begin(worker + 1, total, workers) : 0;
    const uint32_t keys = shared_address(shared) + warp * L::kWarp, values = keys + L::kOperand, queries = values + L::kOperand;
    const int chunk16 = lane % kLanes, sub = lane / kLanes;
    // Byte of 16-byte chunk c of a row: swizzled as in attention_kernel, rows of the head dimension.
    const auto place = [](int row, int c) { return static_cast<uint32_t>(row * kDim * 2 + ((c ^ (row & 7)) << 4)); };
    int continued = -1;
    int group = 0, head = 0;
    if (share < stop) {
        group = static_cast<int>(entry_at(running, groups, share / p.kv_heads));
        const int64_t cost = running[group + 1] - running[group];
        if (cost) head = static_cast<int>((share - static_cast<int64_t>(running[group]) * p.kv_heads) / cost);
    }
    while (share < stop && group < groups) {
        const uint32_t cost = running[group + 1] - running[group];
        const int64_t start = static_cast<int64_t>(running[group]) * p.kv_heads + static_cast<int64_t>(head) * cost;
        if (cost && start >= stop) break;
        const int its_group = group, its_head = head;
        if (!cost || ++head >= p.kv_heads) {
            ++group;
            head = 0;
        }
        if (!cost) continue;
        const int units = item_tiles(cost_unit, cost);
        const int low = first_tile(cost_unit, share, start, units), high = first_tile(cost_unit, stop, start, units);
        if (low >= high) continue;
        if (low) continued = its_group * p.kv_heads + its_head;
        const bool prefix = its_group < offset;
        const int64_t b = its_group - offset;
        Request request{0, p.tokens, 0};
        if (!prefix) request = request_at(p, b);
        const int rows = static_cast<int>(request.fresh) * p.group;
        int table_row;
        if (prefix) {
            table_row = static_cast<int>(p.source_row);
        } else {
            const int64_t at = p.rows ? load_index(p.rows, p.rows_es, b) : b;
            table_row = at >= 0 && at < p.table_rows ? static_cast<int>(at) : -1;
        }
        const int end = prefix ? p.shared : static_cast<int>(request.length < reach ? request.length : reach);
        const int begin = prefix ? 0 : p.shared;
        const int from = begin + low * kFewTile, to = begin + high * kFewTile < end ? begin + high * kFewTile : end;
        const char* k_plane = static_cast<const char*>(p.k_plane) + 2 * its_head * p.k_head + 16 * chunk16;
        const char* v_plane = static_cast<const char*>(p.v_plane) + 2 * its_head * p.v_head + 16 * chunk16;
        const auto find = [&](int position) {
            const int mine = position + lane;
            return look_up(p, lane < kChunk && mine < to ? table_row : -1, static_cast<uint32_t>(mine));
        };
        const auto copy = [&](uint32_t operand, const char* plane, int64_t stride, int slots) {
#pragma unroll
            for (int i = 0; i < kChunk; i += kAtOnce) {
                const int slot = __shfl_sync(0xffffffffu, slots, i + sub);
                copy16_async(operand + place(i + sub, chunk16), slot >= 0 ? plane + slot * stride : static_cast<const char*>(p.query),
                             slot >= 0 ? 16 : 0);
            }
        };
        // Queries and the first chunk.
        for (int i = sub; i < rows; i += kAtOnce) {
            const int token = i / p.group;
            copy16_async(queries + place(i, chunk16),
                         static_cast<const char*>(p.query) + 16 * chunk16 +
                             2 * ((request.begin + token) * p.q_token + (its_head * p.group + i - token * p.group) * p.q_head), 16);
        }
        int slots = slot_of(p, find(from));
        uint32_t there = __ballot_sync(0xffffffffu, slots >= 0);
        copy(keys, k_plane, 2 * p.k_slot, slots);
        copies_commit();
        copy(values, v_plane, 2 * p.v_slot, slots);
        copies_commit();
        // Per row of this lane (two of each block of 8): positions it sees, maximum, sum, output.
        const auto work = [&](auto row_blocks) {
            constexpr int kRowBlocks = decltype(row_blocks)::value;
            int sees[kRowBlocks][2];
            float top[kRowBlocks][2], sum[kRowBlocks][2], out[kDim / 16][kRowBlocks][4];
#pragma unroll
            for (int n = 0; n < kRowBlocks; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = n * 8 + (lane & 3) * 2 + j, token = row / p.group;
                    int64_t seen = 0;
                    if (row < rows) {
                        seen = request.length - request.fresh + token + 1;
                        if (prefix) {
                            int64_t its;
                            Request r;
                            seen = request_of(p, token, its, r) ? r.length - r.fresh + (token - r.begin) + 1 : 0;
                        }
                    }
                    sees[n][j] = seen < 0 ? 0 : static_cast<int>(seen < INT32_MAX ? seen : INT32_MAX);
                    top[n][j] = -INFINITY;
                    sum[n][j] = 0.f;
                }
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) out[d][n][0] = out[d][n][1] = out[d][n][2] = out[d][n][3] = 0.f;
            }
            const int block = lane >> 3, line = lane & 7;  // this lane's address in a load of four 8 x 8 blocks
#pragma unroll 1
            for (int position = from; position < to; position += kChunk) {
                const bool more = position + kChunk < to;
                Lookup next{-1, 0};
                if (more) next = find(position + kChunk);
                copies_wait<1>();  // the keys (and queries)
                __syncwarp();
                float score[kBlocks][kRowBlocks][4] = {};
#pragma unroll
                for (int k = 0; k < kDim / 16; k += 2) {
                    uint32_t q[2][4];
                    if (kRowBlocks == 1) {  // rows 0-7, four chunks of 8 dimensions: two steps
                        load_blocks<false>(queries + place(line, 2 * k + block), q[0]);
                    } else {  // rows 0-7 and 8-15, two chunks: a step each
                        load_blocks<false>(queries + place((block >> 1) * 8 + line, 2 * k + (block & 1)), q[0]);
                        load_blocks<false>(queries + place((block >> 1) * 8 + line, 2 * k + 2 + (block & 1)), q[1]);
                    }
#pragma unroll
                    for (int step = 0; step < 2; ++step) {
#pragma unroll
                        for (int m = 0; m < kBlocks; ++m) {
                            uint32_t a[4];
                            load_blocks<false>(keys + place(m * 16 + (block & 1) * 8 + line, 2 * (k + step) + (block >> 1)), a);
                            if (kRowBlocks == 1) {
                                mma_warp<Kind<T>::kBf16>(score[m][0], a, q[0][2 * step], q[0][2 * step + 1]);
                            } else {
#pragma unroll
                                for (int n = 0; n < kRowBlocks; ++n) {
                                    mma_warp<Kind<T>::kBf16>(score[m][n], a, q[step][2 * n], q[step][2 * n + 1]);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
                const uint32_t seen_now = there;
                if (more) {
                    slots = slot_of(p, next);
                    there = __ballot_sync(0xffffffffu, slots >= 0);
                    copy(keys, k_plane, 2 * p.k_slot, slots);
                }
                copies_commit();
                // A lane's scores: positions lane / 4 and lane / 4 + 8 of each block, two rows.
                float most[kRowBlocks][2];
                bool raise = false;
#pragma unroll
                for (int n = 0; n < kRowBlocks; ++n) {
                    most[n][0] = most[n][1] = -INFINITY;
#pragma unroll
                    for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = m * 16 + (lane >> 2) + (i >> 1) * 8;
                            const bool visible = (seen_now >> at & 1u) && position + at < sees[n][i & 1];
                            score[m][n][i] = visible ? __fmul_rn(score[m][n][i], p.scale_log2) : -INFINITY;
                            most[n][i & 1] = fmaxf(most[n][i & 1], score[m][n][i]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) most[n][j] = fmaxf(most[n][j], __shfl_xor_sync(0xffffffffu, most[n][j], d));
                        raise |= most[n][j] - top[n][j] > kRaise;
                    }
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int n = 0; n < kRowBlocks; ++n) {
                        float factor[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float higher = fmaxf(top[n][j], most[n][j]);
                            factor[j] = top[n][j] == -INFINITY ? 0.f : exp2_approx(top[n][j] - higher);
                            top[n][j] = higher;
                            sum[n][j] *= factor[j];
                        }
#pragma unroll
                        for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) out[d][n][i] *= factor[i & 1];
                        }
                    }
                }
                uint32_t weights[kBlocks][kRowBlocks][2];
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
#pragma unroll
                    for (int n = 0; n < kRowBlocks; ++n) {
                        float w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float base = top[n][i & 1] == -INFINITY ? 0.f : top[n][i & 1];
                            w[i] = exp2_approx(score[m][n][i] - base + Kind<T>::kShift);
                            sum[n][i & 1] += w[i];
                        }
                        weights[m][n][0] = transpose_block(Kind<T>::pack(w[0], w[1]));
                        weights[m][n][1] = transpose_block(Kind<T>::pack(w[2], w[3]));
                    }
                }
                copies_wait<1>();  // the values
                __syncwarp();
#pragma unroll
                for (int d = 0; d < kDim / 16; ++d) {
#pragma unroll
                    for (int m = 0; m < kBlocks; ++m) {
                        uint32_t a[4];
                        load_blocks<true>(values + place(m * 16 + (block >> 1) * 8 + line, 2 * d + (block & 1)), a);
#pragma unroll
                        for (int n = 0; n < kRowBlocks; ++n) {
                            mma_warp<Kind<T>::kBf16>(out[d][n], a, weights[m][n][0], weights[m][n][1]);
                        }
                    }
                }
                __syncwarp();
                if (more) copy(values, v_plane, 2 * p.v_slot, slots);
                copies_commit();
            }
            float* partial = p.few_out + static_cast<int64_t>(worker) * p.few_rows * kDim;
            float2* stat = p.few_stat + static_cast<int64_t>(worker) * p.few_rows;
            if (low == 0) {
                const int64_t row = static_cast<int64_t>(its_head) * p.head_rows + request.begin * p.group;
                partial = (prefix ? p.prefix_out : p.own_out) + row * kDim;
                stat = (prefix ? p.prefix_stat : p.own_stat) + row;
            }
#pragma unroll
            for (int n = 0; n < kRowBlocks; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = n * 8 + (lane & 3) * 2 + j;
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) sum[n][j] += __shfl_xor_sync(0xffffffffu, sum[n][j], d);
                    if (row >= rows) continue;
                    float* target = partial + static_cast<int64_t>(row) * kDim + (lane >> 2);
#pragma unroll
                    for (int d = 0; d < kDim / 16; ++d) {
                        target[16 * d] = out[d][n][j];
                        target[16 * d + 8] = out[d][n][2 + j];
                    }
                    if (lane < 4) stat[row] = make_float2(top[n][j], sum[n][j]);
                }
            }
        };
        if (rows <= 8) {
            work(std::integral_constant<int, 1>{});
        } else {
            work(std::integral_constant<int, 2>{});
        }
        copies_wait_all();
        __syncwarp();
    }
    if (lane == 0 && worker < workers) p.few_next[worker] = continued;
    if (p.large) grid_dependency_wait();  // this grid completes after attention_kernel, so what follows it may read both
}

// ---------------------------------------------------------------- joining the parts

constexpr int kJoinWarps = 4;
constexpr int kJoinLanes = 8;  // of a row

__device__ __forceinline__ bool finite(const float4& v) {
    return isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w);
}

template <typename T, int kDim>
__device__ __forceinline__ void write_row(const AttentionParams& p, int n, int head, int lane, const float4* acc, float scale) {
    T* o = static_cast<T*>(p.out) + n * p.o_token + head * p.o_head + 4 * lane;
#pragma unroll
    for (int v = 0; v < kDim / (4 * kJoinLanes); ++v) {
        *reinterpret_cast<uint2*>(o + v * 4 * kJoinLanes) = make_uint2(Kind<T>::pack(acc[v].x * scale, acc[v].y * scale),
                                                                       Kind<T>::pack(acc[v].z * scale, acc[v].w * scale));
    }
}

// The table row behind the shared positions, -1 for none; the slot of position j.
__device__ __forceinline__ int own_row_of(const AttentionParams& p, int64_t b) {
    const int64_t row = p.rows ? load_index(p.rows, p.rows_es, b) : b;
    return row >= 0 && row < p.table_rows ? static_cast<int>(row) : -1;
}
__device__ __forceinline__ int slot_at(const AttentionParams& p, int own_row, int64_t j) {
    return slot_of(p, look_up(p, j < p.shared ? static_cast<int>(p.source_row) : own_row, static_cast<uint32_t>(j)));
}

// Positions that query token n sees.
__device__ __forceinline__ int64_t seen_by(const AttentionParams& p, const Request& request, int n) {
    const int64_t reach = p.table_width * p.page_size, seen = request.length - request.fresh + 1 + n - request.begin;
    return seen < 0 ? 0 : (seen < reach ? seen : reach);
}

// A row whose weights are all 0 sees no position with a slot (its result is 0), or its scores are all minus infinity (0 / 0).
__device__ __noinline__ bool sees_any(const AttentionParams& p, int64_t b, const Request request, int n) {
    const int lane = static_cast<int>(lane_id()) % kJoinLanes;
    const uint32_t eight = 0xffu << (lane_id() & ~7u);
    const int64_t seen = seen_by(p, request, n);
    const int own_row = own_row_of(p, b);
    bool found = false;
    for (int64_t j = 0; j < seen && !found; j += kJoinLanes) {
        found = __any_sync(eight, j + lane < seen && slot_at(p, own_row, j + lane) >= 0);
    }
    return found;
}

// A weight of 0 does not keep an infinity or NaN out of a product: a V row that a query row does not see
// but another of its tile does (a later token of its request, a shared position behind a short request) may
// leave one in its sum.  Such a row is summed again over the positions it sees, by the eight lanes that join it;
// its maximum and sum stand, they come from the scores alone (`scale` is one over the sum, without kFactor).  False, and nothing is written, if what it does not
// see is finite.  Its query is read before its output is written: they may be the same memory.
template <typename T, int kDim>
__device__ __noinline__ bool sum_again(const AttentionParams& p, int64_t b, const Request request, int n, int head, float top,
                                       float scale) {
    constexpr int kVectors = kDim / (4 * kJoinLanes);
    const int lane = static_cast<int>(lane_id()) % kJoinLanes;
    const uint32_t eight = 0xffu << (lane_id() & ~7u);
    const int kv_head = head / p.group;
    const int64_t at = n - request.begin, reach = p.table_width * p.page_size, seen = seen_by(p, request, n);
    const int64_t row_tile = (at * p.group + head - kv_head * p.group) / (2 * kRows);
    int64_t last = request.length - request.fresh + 1 + last_token(row_tile, request.fresh, p.group);
    if (last > reach) last = reach;
    if (last < p.shared) last = p.shared;
    const int own_row = own_row_of(p, b);
    const auto load = [&](const void* plane, int64_t offset, float4* to) {
        const T* from = static_cast<const T*>(plane) + offset + 4 * lane;
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const uint2 raw = *reinterpret_cast<const uint2*>(from + v * 4 * kJoinLanes);
            const float2 low = Kind<T>::unpack(raw.x), high = Kind<T>::unpack(raw.y);
            to[v] = make_float4(low.x, low.y, high.x, high.y);
        }
    };
    float4 row[kVectors];
    bool found = false;
    for (int64_t j = seen; j < last && !found; ++j) {
        const int slot = slot_at(p, own_row, j);
        if (slot < 0) continue;
        load(p.v_plane, slot * p.v_slot + kv_head * p.v_head, row);
        bool odd = false;
#pragma unroll
        for (int v = 0; v < kVectors; ++v) odd |= !finite(row[v]);
        found = __any_sync(eight, odd);
    }
    if (!found) return false;
    float4 query[kVectors], acc[kVectors];
    load(p.query, n * p.q_token + head * p.q_head, query);
#pragma unroll
    for (int v = 0; v < kVectors; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int64_t j = 0; j < seen; ++j) {
        const int slot = slot_at(p, own_row, j);
        if (slot < 0) continue;
        load(p.k_plane, slot * p.k_slot + kv_head * p.k_head, row);
        float score = 0.f;
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            score += query[v].x * row[v].x + query[v].y * row[v].y + query[v].z * row[v].z + query[v].w * row[v].w;
        }
#pragma unroll
        for (int d = 1; d < kJoinLanes; d <<= 1) score += __shfl_xor_sync(eight, score, d);
        const float weight = exp2_approx(__fmul_rn(score, p.scale_log2) - top);
        load(p.v_plane, slot * p.v_slot + kv_head * p.v_head, row);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            acc[v].x = fmaf(weight, row[v].x, acc[v].x);
            acc[v].y = fmaf(weight, row[v].y, acc[v].y);
            acc[v].z = fmaf(weight, row[v].z, acc[v].z);
            acc[v].w = fmaf(weight, row[v].w, acc[v].w);
        }
    }
    write_row<T, kDim>(p, n, head, lane, acc, scale);
    return true;
}

// Eight lanes a row: the parts (m_i, l_i, O_i) of a row join as
// sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i with m = max m_i.  The blocks (or workers) that may hold a part
// of an item lie next to each other: a lane looks at each, first those of the row's prefix item, then
// those of its own.  Bound by instructions for many rows (eight lanes a row take a quarter of what a warp
// a row takes: 8 prompts of up to 400 tokens, 51,000 rows, 20 us against 42); by the latency of dependent loads for few, so
// then the four eights of a warp (kSplit) share one row's parts and join at the end.  Many rows: six blocks an
// SM (eight, with less than 64 registers a thread, took 2 us more for 8192 rows of 128 requests).
template <typename T, int kDim, int kSplit>
__global__ void __launch_bounds__(32 * kJoinWarps, kSplit == 1 ? 6 : 1) combine_kernel(const __grid_constant__ AttentionParams p) {
    constexpr int kVectors = kDim / (4 * kJoinLanes);  // of four values, of a row, in a lane
    constexpr int kAtOnce = kSplit == 1 ? 2 : 4;       // parts whose loads are on their way together
    constexpr uint32_t kAll = 0xffffffffu;
    const int lane = static_cast<int>(lane_id()) % kJoinLanes;
    const int mine_of = static_cast<int>(threadIdx.x) / kJoinLanes % kSplit;
    const int64_t index = (static_cast<int64_t>(blockIdx.x) * 32 * kJoinWarps + threadIdx.x) / (kJoinLanes * kSplit);
    const int heads = p.kv_heads * p.group;
    const int n = static_cast<int>(index / heads), head = static_cast<int>(index - static_cast<int64_t>(n) * heads);
    const int kv_head = head / p.group, head_row = n * p.group + head - kv_head * p.group;
    int64_t b;
    Request request{0, 0, 0};
    // The requests are as the kernels before found them (they have waited for what writes them).
    const bool active = request_of(p, n, b, request);
    grid_dependency_wait();
    allow_dependents();
    int prefix_item = 0, own_item = 0, local = 0, prefix_first = 0, own_first = 0, prefix_count = 0, count = 0;
    bool few = false;
    if (active) {
        const int prefix_items = p.prefix_tiles ? p.prefix_row_tiles * p.kv_heads : 0;
        few = p.few_own && request.fresh * p.group <= kFewRows;
        local = head_row - static_cast<int>(request.begin) * p.group;
        uint32_t prefix_span = 1, own_span = 1;
        if (p.few_prefix) {
            prefix_item = kv_head;
            prefix_span = p.few_span[prefix_item];
        } else if (prefix_items) {
            prefix_item = kv_head * p.prefix_row_tiles + head_row / (2 * kRows);
            prefix_span = p.item_span[prefix_item];
        }
        if (few) {
            own_item = (static_cast<int>(b) + p.few_prefix) * p.kv_heads + kv_head;
            own_span = p.few_span[own_item];
        } else if (p.large) {
            const int entry = static_cast<int>(p.first_entry[b]) + local / (2 * kRows);
            own_item = prefix_items + entry * p.kv_heads + kv_head;
            if (entry < kMaxEntries) own_span = p.item_span[own_item];
        }
        prefix_first = static_cast<int>(prefix_span & 0xffff);
        own_first = static_cast<int>(own_span & 0xffff);
        prefix_count = static_cast<int>(prefix_span >> 16) - prefix_first + 1;
        count = prefix_count + static_cast<int>(own_span >> 16) - own_first + 1;
    }
    float top = -INFINITY, total = 0.f;
    float4 acc[kVectors];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t bad = 0;  // a wait ran out in a block whose part is needed
#pragma unroll 1
    for (int base = mine_of * kJoinLanes; __any_sync(kAll, base < count); base += kSplit * kJoinLanes) {
        const int candidate = base + lane;
        float2 part = make_float2(-INFINITY, 0.f);
        uint32_t source = 0;  // all parts lie in one workspace: its row of kDim
        if (candidate < count) {
            const bool is_prefix = candidate < prefix_count;
            const bool worker = is_prefix ? p.few_prefix : few;
            const int place = is_prefix ? candidate : candidate - prefix_count;
            const int block = (is_prefix ? prefix_first : own_first) + place;
            const float2* stat;
            const float* values;
            int64_t row;
            bool here = true;
            if (place == 0) {
                row = static_cast<int64_t>(kv_head) * p.head_rows + head_row;
                stat = is_prefix ? p.prefix_stat : p.own_stat;
                values = is_prefix ? p.prefix_out : p.own_out;
            } else {
                const int its_row = is_prefix ? head_row : local;
                row = worker ? static_cast<int64_t>(block) * p.few_rows + its_row
                             : static_cast<int64_t>(block) * 2 * kRows + its_row % (2 * kRows);
                stat = worker ? p.few_stat : p.next_stat;
                values = worker ? p.few_out : p.next_out;
                here = (worker ? p.few_next : p.next_item)[block] == (is_prefix ? prefix_item : own_item);
            }
            const float2 its = stat[row];
            if (here) part = its;
            if (!worker) bad |= p.failed[block];
            source = static_cast<uint32_t>((values - p.prefix_out) / kDim + row);
        }
        const bool counts = part.y != 0.f;  // a sum of 0: the row sees nothing there
        float higher = counts ? part.x : -INFINITY;
#pragma unroll
        for (int d = 1; d < kJoinLanes; d <<= 1) higher = fmaxf(higher, __shfl_xor_sync(kAll, higher, d));
        higher = fmaxf(higher, top);
        const float before = top == -INFINITY ? 0.f : exp2_approx(top - higher);
        const float weight = counts ? exp2_approx(part.x - higher) : 0.f;
        float share = weight * part.y;
#pragma unroll
        for (int d = 1; d < kJoinLanes; d <<= 1) share += __shfl_xor_sync(kAll, share, d);
        top = higher;
        total = total * before + share;
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            acc[v] = make_float4(acc[v].x * before, acc[v].y * before, acc[v].z * before, acc[v].w * before);
        }
#pragma unroll 1
        for (int u = 0; u < kJoinLanes && __any_sync(kAll, base + u < count); u += kAtOnce) {
            float4 value[kAtOnce][kVectors];
            float mine[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                mine[i] = __shfl_sync(kAll, weight, u + i, kJoinLanes);
                const uint32_t its = __shfl_sync(kAll, source, u + i, kJoinLanes);
                const float4* from = reinterpret_cast<const float4*>(p.prefix_out) + static_cast<int64_t>(its) * (kDim / 4) + lane;
#pragma unroll
                for (int v = 0; v < kVectors; ++v) {
                    value[i][v] = mine[i] != 0.f ? from[v * kJoinLanes] : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
                for (int v = 0; v < kVectors; ++v) {
                    acc[v].x = fmaf(value[i][v].x, mine[i], acc[v].x);
                    acc[v].y = fmaf(value[i][v].y, mine[i], acc[v].y);
                    acc[v].z = fmaf(value[i][v].z, mine[i], acc[v].z);
                    acc[v].w = fmaf(value[i][v].w, mine[i], acc[v].w);
                }
            }
        }
    }
#pragma unroll
    for (int d = 1; d < kJoinLanes * kSplit; d <<= 1) bad |= __shfl_xor_sync(kAll, bad, d);
    if (kSplit > 1) {
        float higher = top;
#pragma unroll
        for (int d = kJoinLanes; d < 32; d <<= 1) higher = fmaxf(higher, __shfl_xor_sync(kAll, higher, d));
        const float weight = top == -INFINITY ? 0.f : exp2_approx(top - higher);
        top = higher;
        total *= weight;
#pragma unroll
        for (int d = kJoinLanes; d < 32; d <<= 1) total += __shfl_xor_sync(kAll, total, d);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            float* a = reinterpret_cast<float*>(&acc[v]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] *= weight;
#pragma unroll
                for (int d = kJoinLanes; d < 32; d <<= 1) a[i] += __shfl_xor_sync(kAll, a[i], d);
            }
        }
    }
    if (!active || mine_of) return;
    float scale = bad ? NAN : (total == 0.f ? 0.f : 1.f / total);
    if (total == 0.f && sees_any(p, b, request, n)) scale = NAN;
    if (p.lse && lane == 0) {
        p.lse[n * p.lse_token + head * p.lse_head] =
            bad ? NAN : (total == 0.f ? -INFINITY : (top + log2f(total * (1.f / Kind<T>::kFactor))) * 0.69314718055994531f);
    }
    bool odd = false;
#pragma unroll
    for (int v = 0; v < kVectors; ++v) odd |= !finite(acc[v]);
    if (__any_sync(0xffu << (lane_id() & ~7u), odd) && !bad && isfinite(total) &&
        sum_again<T, kDim>(p, b, request, n, head, top, scale * Kind<T>::kFactor)) {
        return;
    }
    write_row<T, kDim>(p, n, head, lane, acc, scale);
}

// ---------------------------------------------------------------- host side

struct Workspace {
    int64_t prefix_out, own_out, next_out, prefix_stat, own_stat, next_stat, item_span, first_entry, next_item, failed;
    int64_t few_out, few_stat, few_span, few_next, bytes;
};

int64_t few_workers(int64_t blocks) { return blocks * 2 * kFewWarps; }

Workspace workspace_of(int64_t tokens, int64_t batch, int64_t query_heads, int64_t kv_heads, int64_t dim, int64_t blocks) {
    Workspace w{};
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 511) / 512 * 512;  // whole rows of any head dimension
        return here;
    };
    const int64_t rows = tokens * query_heads, next = blocks * 2 * kRows;
    w.prefix_out = take(rows * dim * 4);
    w.own_out = take(rows * dim * 4);
    w.next_out = take(next * dim * 4);
    w.prefix_stat = take(rows * 8);
    w.own_stat = take(rows * 8);
    w.next_stat = take(next * 8);
    const int64_t row_tiles = (rows / kv_heads + 2 * kRows - 1) / (2 * kRows);
    w.item_span = take((row_tiles + kMaxEntries) * kv_heads * 4);
    w.first_entry = take(batch * 4);
    w.next_item = take(blocks * 4);
    w.failed = take(blocks * 4);
    const int64_t workers = few_workers(blocks);
    w.few_out = take(workers * kFewRows * dim * 4);
    w.few_stat = take(workers * kFewRows * 8);
    w.few_span = take((batch + 1) * kv_heads * 4);
    w.few_next = take(workers * 4);
    w.bytes = at;
    return w;
}

template <typename T, int kDim>
void launch(const AttentionParams& p, cudaStream_t stream) {
    using L = Layout<kDim>;
    static_assert(L::kBytes <= 232448, "shared memory of one block");
    cuda_check(cudaFuncSetAttribute(attention_kernel<T, kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes),
               "attention shared memory");
    if (p.large) {
        launch_dependent(attention_kernel<T, kDim>, dim3(static_cast<unsigned>(p.blocks)), dim3(kThreads), L::kBytes, stream,
                         "shared_prefix_attention launch", p);
    }
    if (p.few_prefix || p.few_own) {
        constexpr uint32_t kFewBytes = FewLayout<kDim>::kBytes;
        cuda_check(cudaFuncSetAttribute(rows_kernel<T, kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewBytes),
                   "attention shared memory");
        launch_dependent(rows_kernel<T, kDim>, dim3(static_cast<unsigned>(p.workers / kFewWarps)), dim3(32 * kFewWarps),
                         kFewBytes, stream, "shared_prefix_attention rows", p);
    }
    // A warp a row while all of them fit the GPU at once, a quarter of one behind that.
    const int64_t rows = p.tokens * p.kv_heads * p.group;
    const bool split = rows <= static_cast<int64_t>(p.blocks) * 48;
    const int64_t threads = rows * kJoinLanes * (split ? 4 : 1);
    launch_dependent(split ? combine_kernel<T, kDim, 4> : combine_kernel<T, kDim, 1>,
                     dim3(static_cast<unsigned>((threads + 32 * kJoinWarps - 1) / (32 * kJoinWarps))), dim3(32 * kJoinWarps),
                     0, stream, "shared_prefix_attention join", p);
}

void check_shape(int64_t tokens, int64_t batch, int query_heads, int kv_heads, int head_dim) {
    require(tokens >= 0 && batch >= 0, "negative attention dimensions");
    require(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
    require(kv_heads >= 1 && query_heads >= 1 && query_heads % kv_heads == 0,
            "query_heads must be a positive multiple of kv_heads");
    require(query_heads <= 65535, "more than 65535 query heads");
    const int64_t group = query_heads / kv_heads;
    require(batch <= kMaxEntries && tokens <= INT32_MAX / query_heads &&
                batch + (tokens * group + 2 * kRows - 1) / (2 * kRows) <= kMaxEntries,
            "more than EKV_ATTENTION_MAX_ROW_TILES row tiles in one call");
}

}  // namespace
}  // namespace ekv

extern "C" int ekv_shared_prefix_workspace(int64_t tokens, int64_t batch, int query_heads, int kv_heads, int head_dim,
                                           int device, int64_t* bytes) {
    using namespace ekv;
    return guarded([&] {
        require(bytes != nullptr, "null pointer argument");
        check_shape(tokens, batch, query_heads, kv_heads, head_dim);
        *bytes = tokens && batch ? workspace_of(tokens, batch, query_heads, kv_heads, head_dim, sm_count(device)).bytes : 0;
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
        require(slots >= 0 && slots <= INT32_MAX && table_rows >= 0 && table_width >= 0 && tokens >= 0 && batch >= 0,
                "negative attention dimensions, or more than 2^31 - 1 slots");
        require(dtype == EKV_BF16 || dtype == EKV_FP16, "dtype must be EKV_BF16 or EKV_FP16");
        check_shape(tokens, batch, query_heads, kv_heads, head_dim);
        require(page_size >= 1 && page_size <= INT32_MAX, "page_size outside [1, 2^31)");
        // The end of the last tile is held in 32 bits too.
        require(table_width <= (INT32_MAX - 255) / page_size, "a table row covers more than 2^31 - 256 positions");
        require(shared_tokens >= 0 && shared_tokens <= table_width * page_size,
                "shared_tokens outside the table's positions");
        require(!shared_tokens || (source_row >= 0 && source_row < table_rows), "source row is outside the block table");
        // The kernels' factor, scale * log2(e), has to be finite too.
        require(scale > 0.f && scale <= 2.3e38f, "scale must lie in (0, 2.3e38]");
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
        const int group = query_heads / kv_heads;
        const int64_t head_rows = tokens * group;
        // The plan's running cost of one head is held in 32 bits.
        const int64_t most_tiles = (table_width * page_size + kTile - 1) / kTile;
        const int64_t most_entries = batch + (head_rows + 2 * kRows - 1) / (2 * kRows);
        require((most_tiles * kBothTile + kBothStart) <= static_cast<int64_t>(UINT32_MAX) / most_entries,
                "the block table is too wide for this batch");
        bind_device(device);
        const int blocks = sm_count(device);
        const Workspace w = workspace_of(tokens, batch, query_heads, kv_heads, head_dim, blocks);
        require(workspace != nullptr && workspace_bytes >= w.bytes, "workspace is too small");
        require(reinterpret_cast<uint64_t>(workspace) % 256 == 0, "workspace must be 256-byte aligned");
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
        p.page_size = static_cast<uint32_t>(page_size);
        p.page_log2 = -1;
        for (int bit = 0; bit < 31; ++bit) {
            if (page_size == int64_t{1} << bit) p.page_log2 = bit;
        }
        p.tokens = tokens;
        p.batch = batch;
        p.shared = static_cast<int>(shared_tokens);
        p.source_row = source_row;
        p.kv_heads = kv_heads;
        p.group = group;
        p.table_es = table_esize;
        p.rows_es = rows_esize;
        p.len_es = lengths_esize;
        p.starts_es = starts_esize;
        p.scale_log2 = scale * 1.4426950408889634f;
        p.head_rows = static_cast<int>(head_rows);
        p.prefix_row_tiles = static_cast<int>((head_rows + 2 * kRows - 1) / (2 * kRows));
        p.prefix_tiles = static_cast<int>((shared_tokens + kTile - 1) / kTile);
        p.blocks = blocks;
        p.workers = static_cast<int>(few_workers(blocks));
        p.few_own = group <= kFewRows;
        p.few_rows = static_cast<int>(head_rows < kFewRows ? head_rows : kFewRows);
        if (!query_starts && !(shared_tokens && head_rows <= kFewRows)) p.few_rows = group < kFewRows ? group : kFewRows;
        p.few_prefix = shared_tokens > 0 && head_rows <= kFewRows && shared_tokens <= kFewPrefix;
        if (p.few_prefix) p.prefix_tiles = 0;
        // With one token a request, all of them have `group` rows.
        p.large = p.prefix_tiles > 0 || (query_starts ? head_rows > kFewRows : !p.few_own);
        char* at = static_cast<char*>(workspace);
        p.prefix_out = reinterpret_cast<float*>(at + w.prefix_out);
        p.own_out = reinterpret_cast<float*>(at + w.own_out);
        p.next_out = reinterpret_cast<float*>(at + w.next_out);
        p.prefix_stat = reinterpret_cast<float2*>(at + w.prefix_stat);
        p.own_stat = reinterpret_cast<float2*>(at + w.own_stat);
        p.next_stat = reinterpret_cast<float2*>(at + w.next_stat);
        p.item_span = reinterpret_cast<uint32_t*>(at + w.item_span);
        p.first_entry = reinterpret_cast<uint32_t*>(at + w.first_entry);
        p.next_item = reinterpret_cast<int*>(at + w.next_item);
        p.few_out = reinterpret_cast<float*>(at + w.few_out);
        p.few_stat = reinterpret_cast<float2*>(at + w.few_stat);
        p.few_span = reinterpret_cast<uint32_t*>(at + w.few_span);
        p.few_next = reinterpret_cast<int*>(at + w.few_next);
        p.failed = reinterpret_cast<uint32_t*>(at + w.failed);
        const auto cstream = static_cast<cudaStream_t>(stream);
        if (dtype == EKV_BF16) {
            head_dim == 128 ? launch<__nv_bfloat16, 128>(p, cstream)
                            : launch<__nv_bfloat16, 64>(p, cstream);
        } else {
            head_dim == 128 ? launch<__half, 128>(p, cstream) : launch<__half, 64>(p, cstream);
        }
        check_launch("shared_prefix_attention launch");
    });
}
