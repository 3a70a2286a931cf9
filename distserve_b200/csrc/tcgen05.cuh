// Thin wrappers of the 5th-generation tensor core's instructions (sm_100a): tensor memory, matrix products issued by one
// thread, and the barriers that order them with ordinary code.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace kvmig {

// ---- barriers in shared memory ---------------------------------------------------------------------------

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool barrier_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

constexpr unsigned kWaitPolls = 1u << 26;
constexpr unsigned long long kWaitNs = 2000000000ull;

// Waits for a phase, for two seconds at most or until another thread of the block has given up (*failed).
__device__ __forceinline__ bool barrier_wait_slow(uint32_t bar, uint32_t parity, volatile int* failed) {
    unsigned long long t0, t;
    if (*failed) return false;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (unsigned i = 0; i < kWaitPolls; ++i) {
        if (barrier_test(bar, parity)) return true;
        if ((i & 63u) == 63u) {
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
            if (*failed || t - t0 > kWaitNs) break;
        }
    }
    *failed = 1;
    return false;
}
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
    if (barrier_test(bar, parity)) return true;
    return barrier_wait_slow(bar, parity, failed);
}

// A whole warp waits, and goes on or gives up together.
__device__ __forceinline__ bool barrier_wait_warp(uint32_t bar, uint32_t parity, volatile int* failed) {
    return __all_sync(0xffffffffu, barrier_wait(bar, parity, failed)) != 0;
}

// Makes this thread's writes to shared memory visible to the tensor core and the copy engine.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- copy engine: to shared memory, completing on a barrier ------------------------------------------------

__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Addresses and sizes are multiples of 16 bytes.
__device__ __forceinline__ void bulk_copy(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const void* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// A box of a tensor; x * element size is a multiple of 16 bytes.
__device__ __forceinline__ void box_copy(uint32_t to, const void* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void box_copy(uint32_t to, const void* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

// ---- tensor memory ---------------------------------------------------------------------------------------

// One warp allocates; the address is left in shared memory.
__device__ __forceinline__ void tmem_alloc(uint32_t to, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define KVMIG_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define KVMIG_X8(x, i) "+r"(x[i]), "+r"(x[i + 1]), "+r"(x[i + 2]), "+r"(x[i + 3]), "+r"(x[i + 4]), "+r"(x[i + 5]), "+r"(x[i + 6]), "+r"(x[i + 7])
#define KVMIG_W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])

// 32 columns of the lane's row; the values are there when this returns.
__device__ __forceinline__ void tmem_load(uint32_t (&x)[32], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : KVMIG_R8(x, 0), KVMIG_R8(x, 8), KVMIG_R8(x, 16), KVMIG_R8(x, 24) : "r"(at) : "memory");
}
// 64 columns; the values are there after tmem_wait(x).
__device__ __forceinline__ void tmem_load_async(uint32_t (&x)[64], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,"
        "%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
        : KVMIG_R8(x, 0), KVMIG_R8(x, 8), KVMIG_R8(x, 16), KVMIG_R8(x, 24), KVMIG_R8(x, 32), KVMIG_R8(x, 40), KVMIG_R8(x, 48), KVMIG_R8(x, 56)
        : "r"(at) : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&x)[64]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : KVMIG_X8(x, 0), KVMIG_X8(x, 8), KVMIG_X8(x, 16), KVMIG_X8(x, 24), KVMIG_X8(x, 32), KVMIG_X8(x, 40), KVMIG_X8(x, 48), KVMIG_X8(x, 56)
                 :: "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t at, const uint32_t (&x)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at), KVMIG_W8(x, 0), KVMIG_W8(x, 8), KVMIG_W8(x, 16), KVMIG_W8(x, 24) : "memory");
}
#undef KVMIG_R8
#undef KVMIG_X8
#undef KVMIG_W8

// ---- products --------------------------------------------------------------------------------------------

// Descriptor of an operand in shared memory, laid out in rows of 128 bytes with the 128-byte swizzle (16-byte piece j of
// row r stands at j ^ (r % 8)), 8 rows to 1024 bytes: `stride` bytes from one 8 rows to the next, and, for operands
// whose rows run along the contraction, `lead` bytes from one 128-byte column of rows to the next.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t lead, uint32_t stride) {
    return (uint64_t)((at & 0x3ffffu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Shape and types of a product of 16-bit operands with 32-bit sums.  across: B's rows run along the contraction.
__host__ __device__ constexpr uint32_t product_kind(bool bf16, int m, int n, bool across, bool negate_a) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (negate_a ? 1u << 13 : 0u) | (across ? 1u << 16 : 0u) |
           (uint32_t)(n / 8) << 17 | (uint32_t)(m / 16) << 24;
}

// d (+)= a b over 16 of the contraction, a from shared memory or from tensor memory.  One thread issues it.
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(kind), "r"((uint32_t)add) : "memory");
}
// One lane of a converged warp, the same one every time.  What it issues sits in warp-uniform control flow, so that the
// compiler can keep descriptors in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
// The barrier receives one arrival when everything that this thread has issued is done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

}  // namespace kvmig
