// What kernels with tensor-core products share: TMA copies, barriers with an end, TMEM, and the matrix instruction (sm_100a).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "waits.h"

namespace ffcvb {

// A map of a matrix [rows, cols] of 16- or 32-bit values, rows `stride` values apart, whose boxes are 128 bytes wide and `box` rows high and lie
// swizzled in shared memory (16-byte piece j of a box's row r is at piece j ^ (r & 7)).  What is outside is read as 0 and not written.
// False where the driver has no such call or refuses the sizes.
bool matrix_map(CUtensorMap *map, int type, const void *at, int64_t rows, int64_t cols, int64_t stride, int box);

#ifdef __CUDACC__

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t nanoseconds() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// The same place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t there(uint32_t at, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
__device__ __forceinline__ void barrier_arrive_there(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_passed(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}
__device__ __forceinline__ bool barrier_wait(Waiter &waiter, uint32_t bar, uint32_t parity) {
    return waiter([&] { return barrier_passed(bar, parity); }, nanoseconds);
}

__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
// By one of a pair of CTAs, whose barrier is the first one's.
__device__ __forceinline__ void copy_box_of_pair(uint32_t to, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x), "r"(y),
                 "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap *map, int x, int y, uint32_t from) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(from) : "memory");
}
__device__ __forceinline__ void add_box(const CUtensorMap *map, int x, int y, uint32_t from) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(from) : "memory");
}
__device__ __forceinline__ void boxes_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void boxes_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void boxes_written() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void shared_to_copies() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// (PAIR, here and below: of both CTAs of a pair, each of which calls these.)
template <bool PAIR> __device__ __forceinline__ void tmem_alloc(uint32_t to, uint32_t columns) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        return;
    }
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <bool PAIR> __device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
        return;
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A matrix operand in shared memory, from boxes of 128 bytes by 8 n rows.  Either a box's rows are the operand's rows and the sum runs along them
// (`across` unused), or they run along the sum and a box has 64 of the operand's rows, the next 64 `across` bytes on.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t across) {
    constexpr uint64_t kEight = 1024 >> 4; // from eight of a box's rows to the next
    return (uint64_t)(at >> 4) | (uint64_t)(across >> 4) << 16 | kEight << 32 | 1ull << 46 | 2ull << 61;
}
// The instruction's sizes and types: products of 16 bits, sums of 32; 128 rows, or a pair's 256.
__device__ __forceinline__ uint32_t product_kind(bool bf16, int rows, int columns, bool a_along_sum, bool b_along_sum) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_along_sum ? 1u << 15 : 0u) | (b_along_sum ? 1u << 16 : 0u) | (uint32_t)(columns >> 3) << 17 | (uint32_t)(rows >> 4) << 24;
}
// One thread multiplies; a pair's first CTA does it for both, which have 128 rows of A and half of B's columns each, in the same places, and get their rows' sums.
template <bool PAIR> __device__ __forceinline__ void multiply(uint32_t tmem, uint64_t a, uint64_t b, uint32_t kind, bool add) {
    if constexpr (PAIR) {
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem), "l"(a), "l"(b), "r"(kind),
                     "r"((uint32_t)add)
                     : "memory");
        return;
    }
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem), "l"(a), "l"(b), "r"(kind),
                 "r"((uint32_t)add)
                 : "memory");
}
// The barrier is arrived at once all multiplications issued so far are done: a pair's, in both CTAs.
template <bool PAIR> __device__ __forceinline__ void when_multiplied(uint32_t bar) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
        return;
    }
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 columns of a warp's 32 rows; a lane gets its row's.  They are there once tmem_wait() has been called for them.
__device__ __forceinline__ void tmem_load(uint32_t (&v)[32], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ float tmem_load_one(uint32_t at) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(v) : "r"(at) : "memory");
    return __uint_as_float(v);
}

#endif

} // namespace ffcvb
