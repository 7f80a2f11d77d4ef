// The instructions of the tensor-core kernels: barriers in shared memory, tensor copies, tcgen05 products, and waits that end.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "floatops.cuh"

namespace zkb {
namespace tc {

__device__ __forceinline__ uint32_t smem_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- barriers ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool barrier_done(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// No wait on a barrier is endless: one that has lasted two seconds (or 2^28 tries) marks the block, and through `flag`, which the host
// reads at every call and whenever it has waited for a stream, the process; every role of the block then leaves its loop.
struct Watch {
    volatile int* dead;   // shared memory, of the block
    int* flag;            // mapped host memory
};
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, const Watch& w, bool draining = false) {
    if (barrier_done(bar, parity)) return true;
    unsigned long long start = 0;
    for (unsigned i = 0; i < (1u << 28); ++i) {
        if (barrier_done(bar, parity)) return true;
        if ((i & 63) != 63) continue;
        if (!draining && *w.dead) return false;
        const unsigned long long t = now_ns();
        if (!start) start = t;
        else if (t - start > 2000000000ull) break;
    }
    *w.dead = 1;
    *reinterpret_cast<volatile int*>(w.flag) = 1;
    return false;
}
// The same by a whole warp, which stays together: instructions on tensor memory follow that all its lanes have to reach as one.
__device__ __forceinline__ bool barrier_wait_warp(uint32_t bar, uint32_t parity, const Watch& w) {
    unsigned long long start = 0;
    for (unsigned i = 0; i < (1u << 28); ++i) {
        if (__all_sync(0xffffffffu, barrier_done(bar, parity))) return true;
        if ((i & 63) != 63) continue;
        const unsigned long long t = now_ns();
        if (!start) start = t;
        if (__any_sync(0xffffffffu, *w.dead || t - start > 2000000000ull)) break;
    }
    *w.dead = 1;
    *reinterpret_cast<volatile int*>(w.flag) = 1;
    __syncwarp();
    return false;
}
// some milliseconds: long after the copies and products that a block has in flight
__device__ __forceinline__ void pause() {
    const unsigned long long start = now_ns();
    for (unsigned i = 0; i < (1u << 20) && now_ns() - start < 10000000ull; ++i) __nanosleep(1000);
}
// The flag that the kernels of this process raise (device and host address the same memory); null and the error text on failure.
int* wait_flag();

// ---- clusters --------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// the same place in the shared memory of another block of the cluster
__device__ __forceinline__ uint32_t address_in(uint32_t address, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(address), "r"(rank));
    return a;
}
__device__ __forceinline__ void barrier_arrive_in(uint32_t cluster_address) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_address) : "memory");
}

// ---- tensor copies ---------------------------------------------------------------------------------------------------------
// [rows, cols] of 16-bit values, rows `ld` values apart, read in boxes of 64 columns (128 bytes, swizzled by 128) and box_rows rows;
// what lies outside reads as zero.  The address and ld * 2 have to be multiples of 16.
int make_map(CUtensorMap* map, int dtype, const void* p, size_t rows, size_t cols, size_t ld, unsigned box_rows);

__device__ __forceinline__ void load_box(const CUtensorMap* m, uint32_t dst, uint32_t bar, int col, int row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(m), "r"(bar),
        "r"(col), "r"(row)
        : "memory");
}

// The same copy by one block of a pair, arriving at a barrier of either (an address of the cluster's shared memory).
__device__ __forceinline__ void load_box_pair(const CUtensorMap* m, uint32_t dst, uint32_t bar, int col, int row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(m),
        "r"(bar), "r"(col), "r"(row)
        : "memory");
}
// `bytes` consecutive bytes; both addresses and the size are multiples of 16
__device__ __forceinline__ void load_bytes(uint32_t dst, unsigned long long src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// ---- tcgen05 -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t at, uint32_t cols) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
    __syncwarp();
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t at, uint32_t cols) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t tmem, uint32_t cols) {
    __syncwarp();
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// arrives at the barrier when the products issued so far by this thread are done
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// the same for products of a pair, at the barriers of this place in both blocks
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// A tile in shared memory, swizzled by 128 bytes.  K-major: rows of 128 bytes (64 values of k), groups of 8 rows 1024 bytes apart.  MN-major: k
// rows of 128 bytes (64 values of m or n), groups of 8 k's 1024 bytes apart, groups of 64 m's or n's `group` bytes apart.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t address, bool mn_major, uint32_t group) {
    const uint64_t leading = mn_major ? group >> 4 : 1, stride = 1024 >> 4;
    return (uint64_t)((address >> 4) & 0x3fff) | leading << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}
template <class T> __host__ __device__ constexpr uint32_t instruction(unsigned m, unsigned n, bool a_mn, bool b_mn) {
    const uint32_t type = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;   // bf16 or f16, sums in f32
    return 1u << 4 | type << 7 | type << 10 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (n >> 3) << 17 | (m >> 4) << 24;
}
__device__ __forceinline__ void product(uint32_t tmem, uint64_t a, uint64_t b, uint32_t instr, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem), "l"(a), "l"(b),
        "r"(instr), "r"((uint32_t)add)
        : "memory");
}
// one product over both blocks of a pair, issued by the first: each block holds half of the rows of a and of d and half of the columns of b
__device__ __forceinline__ void product_pair(uint32_t tmem, uint64_t a, uint64_t b, uint32_t instr, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem), "l"(a), "l"(b),
        "r"(instr), "r"((uint32_t)add)
        : "memory");
}
// 32 columns of this warp's 32 lanes: lane i of the warp gets row i
__device__ __forceinline__ void load_columns(uint32_t tmem, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
        "%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(tmem)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void load_columns16(uint32_t tmem, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(tmem)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

}  // namespace tc
}  // namespace zkb
