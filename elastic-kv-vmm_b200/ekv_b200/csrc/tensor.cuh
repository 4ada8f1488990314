// sm_100a tensor-core, tensor-memory and barrier primitives (inline PTX).
#pragma once

#include "common.cuh"

namespace ekv {

// ---------------------------------------------------------------- mbarriers

__device__ __forceinline__ uint32_t shared_address(const void* pointer) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(pointer));
}

__device__ __forceinline__ void barrier_init(uint32_t barrier, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_arrive(uint32_t barrier) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(barrier) : "memory");
}

// May suspend the thread until the phase is complete, for up to kSuspend nanoseconds.
constexpr uint32_t kSuspend = 1000000;

__device__ __forceinline__ bool barrier_try(uint32_t barrier, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(barrier), "r"(parity), "r"(kSuspend)
        : "memory");
    return done != 0;
}

__device__ __forceinline__ uint64_t device_nanoseconds() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Nanoseconds after which a wait inside a kernel gives up.
constexpr uint64_t kWaitLimit = 4000000000ull;

// Wait for the phase of `parity` to complete.  False (and *failed set) when kWaitLimit passes or
// another thread of the block has given up.  Kept short: a kernel has many waits.
__device__ __forceinline__ bool barrier_wait(uint32_t barrier, uint32_t parity, volatile uint32_t* failed) {
    uint32_t tries = 0;
    uint64_t begin = 0;
#pragma unroll 1
    while (!barrier_try(barrier, parity)) {
        if (++tries & 15) continue;
        const uint64_t now = device_nanoseconds();
        if (!begin) begin = now;
        if (*failed || now - begin > kWaitLimit) {
            *failed = 1;
            return false;
        }
    }
    return true;
}

// A count in shared memory that one thread raises, and a wait until it is at least `target`, bounded as above.
__device__ __forceinline__ void count_store(uint32_t address, uint32_t value) {
    asm volatile("st.release.cta.shared::cta.b32 [%0], %1;" ::"r"(address), "r"(value) : "memory");
}
__device__ __forceinline__ bool count_wait(uint32_t address, uint32_t target, volatile uint32_t* failed) {
    uint64_t begin = 0;
#pragma unroll 1
    while (true) {
        uint32_t value;
        asm volatile("ld.acquire.cta.shared::cta.b32 %0, [%1];" : "=r"(value) : "r"(address) : "memory");
        if (value >= target) return true;
        const uint64_t now = device_nanoseconds();
        if (!begin) begin = now;
        if (*failed || now - begin > kWaitLimit) {
            *failed = 1;
            return false;
        }
    }
}

// ---------------------------------------------------------------- proxies and asynchronous copies

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 16 bytes global -> shared; zeros when `bytes` is 0 (then nothing is read).
__device__ __forceinline__ void copy16_async(uint32_t target, const void* source, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(target), "l"(source), "r"(bytes) : "memory");
}
// One arrival at `barrier` (counted in advance) when this thread's copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint32_t barrier) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(barrier) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last kPending groups have landed.
template <int kPending>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void copies_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Registers a thread may use from here on (all warps of the warpgroup together).
template <int kRegisters>
__device__ __forceinline__ void registers_grow() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
template <int kRegisters>
__device__ __forceinline__ void registers_shrink() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters));
}

// ---------------------------------------------------------------- tensor memory

__device__ __forceinline__ void tensor_alloc(uint32_t shared_slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_slot), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tensor_free(uint32_t address, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define EKV_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define EKV_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])

// This lane's 32 consecutive columns (the warp's 32 lanes are tensor-memory lanes).
__device__ __forceinline__ void tensor_load32(uint32_t address, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : EKV_R8(r, 0), EKV_R8(r, 8), EKV_R8(r, 16), EKV_R8(r, 24)
        : "r"(address));
}
__device__ __forceinline__ void tensor_load16(uint32_t address, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : EKV_R8(r, 0), EKV_R8(r, 8)
        : "r"(address));
}
__device__ __forceinline__ void tensor_store16(uint32_t address, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::EKV_I8(
            r, 0),
        EKV_I8(r, 8), "r"(address)
        : "memory");
}

// 32 bytes (a whole sector) to a 32-byte aligned address.
__device__ __forceinline__ void store_sector(float* target, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(target), EKV_I8(r, 0) : "memory");
}

// ---------------------------------------------------------------- matrix products

// Instruction descriptor of a 16-bit product with 32-bit accumulation (M x N).
__host__ __device__ constexpr uint32_t mma_descriptor(bool bf16, int m, int n, bool b_rows_are_k) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_rows_are_k ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// Shared-memory operand of 128-byte rows, swizzled by 128 bytes, in blocks of 8 rows (1024
// bytes).  `block_stride`: bytes from one 128-byte wide column block to the next (used where a
// row of 128 bytes runs along the operand's outer dimension).
__device__ __forceinline__ uint64_t shared_operand(uint32_t address, uint32_t block_stride) {
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (static_cast<uint64_t>(block_stride >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t descriptor, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(descriptor), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// The left operand in tensor memory (two 16-bit values to a column).
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t descriptor, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(descriptor), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// One arrival at `barrier` when every product this thread has issued is complete.
__device__ __forceinline__ void mma_commit(uint32_t barrier) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
}

// ---------------------------------------------------------------- products of one warp

// Four 8 x 8 blocks of 16-bit values, a row's address from each lane; transposed with kTranspose.
template <bool kTranspose>
__device__ __forceinline__ void load_blocks(uint32_t address, uint32_t (&r)[4]) {
    if (kTranspose) {
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(address)
                     : "memory");
    } else {
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(address)
                     : "memory");
    }
}
__device__ __forceinline__ uint32_t transpose_block(uint32_t r) {
    uint32_t t;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(r));
    return t;
}
// c (16 x 8, 32 bits) += a (16 x 16) b (16 x 8).
template <bool kBf16>
__device__ __forceinline__ void mma_warp(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (kBf16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 w, x, y;\n"
        " mov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

}  // namespace ekv
