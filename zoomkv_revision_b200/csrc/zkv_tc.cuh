// zkv_tc.cuh -- 5th-generation tensor cores (tcgen05): tensor memory, shared
// memory and instruction descriptors, waits and loads, as inline PTX.
#pragma once

#include "zkv_common.cuh"

namespace zkv {
namespace tc {

constexpr uint64_t kWaitNs = 2000000000ull;  // longest wait of a kernel on its own copies and products

// One lane of a whole warp, always the same.  Copies and products are issued under it in code that the whole warp runs:
// their operands live in uniform registers, and under a test of the lane number the compiler moves them there for each.
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// Wait for a phase, at most kWaitNs; false and ZKV_ERR_TIMEOUT on expiry.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, int32_t* status) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try(bar, parity)) {
        if (globaltimer_ns() - t0 > kWaitNs) {
            if (status) atomicMax(status, ZKV_ERR_TIMEOUT);
            return false;
        }
    }
    return true;
}

// The same for a whole warp, which goes on together.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, int32_t* status) {
    return __all_sync(0xffffffffu, wait_for(bar, parity, status));
}

__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// A tile of a 2-D tensor map [rows][128-byte columns]: x in bytes, a multiple of 128.
__device__ __forceinline__ void tma_2d(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
// The tile into L2 only: it may be asked for before an earlier kernel has ended, as L2 is where its writes go too.
__device__ __forceinline__ void prefetch_3d(const void* map, int x, int y, int z) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(map), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const void* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ------------------------------------------------------------ pairs
// Two CTAs of a cluster whose tensor cores work on one tile; rank 0 leads.
// Copies and arrivals on barriers of the other CTA.
// The arrival publishes nothing but that tensor memory has been read, which the tcgen05 fences order: a release at cluster
// scope waits for the thread's outstanding accesses of every kind and made a block of the inner dimension take 2400
// clocks instead of 1000 (4096 x 6144 x 4096: 217 us, 104 without).
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {  // an address of in_cta()
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Into this CTA's memory, counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_3d_pair(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t to, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t at, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
// Arrives on the barrier at the same place in both CTAs.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar)
        : "memory");
}
// D[256][n] = A[256][32] B[n][32]^T: each CTA holds 128 rows of A and D, and half of B's rows.
__device__ __forceinline__ void mma_e4m3_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool more) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(desc), "r"((uint32_t)more)
        : "memory");
}

// ------------------------------------------------------------ stores
// A tile in shared memory (128-byte rows, swizzled) to a tensor map; the caller has fenced its writes (fence_async).
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tma_store_2d(const void* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x),
                 "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ------------------------------------------------------------ single words
// 4 bytes from global to shared memory, without a register; `in` false: a zero.
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// This thread's arrival on `bar`, once its copies issued so far have landed.
__device__ __forceinline__ void copy4_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void copy4_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ------------------------------------------------------------ tensor memory
// 128 lanes x 512 columns of 32 bits an SM.  alloc and free by one whole warp.
template <int kColumns>
__device__ __forceinline__ void tmem_alloc(uint32_t to) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "n"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int kColumns>
__device__ __forceinline__ void tmem_free(uint32_t at) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(kColumns) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Until this thread's loads have landed.  The registers are named, so that no use of them is moved before it.
template <int N>
__device__ __forceinline__ void wait_ld(uint32_t (&r)[N]) {
    static_assert(N == 16 || N == 32, "the loads below");
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
    if (N == 32)
        asm volatile(""
                     : "+r"(r[N - 16]), "+r"(r[N - 15]), "+r"(r[N - 14]), "+r"(r[N - 13]), "+r"(r[N - 12]), "+r"(r[N - 11]),
                       "+r"(r[N - 10]), "+r"(r[N - 9]), "+r"(r[N - 8]), "+r"(r[N - 7]), "+r"(r[N - 6]), "+r"(r[N - 5]),
                       "+r"(r[N - 4]), "+r"(r[N - 3]), "+r"(r[N - 2]), "+r"(r[N - 1])::"memory");
}

// Arrives on `bar` when the products issued by this thread so far are done.
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 16 columns of the warp's 32 lanes: thread = lane, register = column.
__device__ __forceinline__ void ld(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}

// 32 columns of the warp's 32 lanes.
__device__ __forceinline__ void ld(uint32_t at, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}

// ------------------------------------------------------------ products
// A tile of rows of 128 bytes, rows one after the other, in the 128-byte
// swizzle that the tensor map writes: groups of 8 rows are 1024 bytes apart.
// `at` 1024-byte aligned, plus 32 bytes for each step of 32 along the row.
__device__ __forceinline__ uint64_t tile_desc(uint32_t at) {
    return (uint64_t)((at & 0x3ffffu) >> 4) | (1ull << 16) | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// e4m3 x e4m3 -> fp32, both operands with the inner dimension contiguous.
__host__ __device__ constexpr uint32_t e4m3_desc(int m, int n) {
    return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// D[m][n] (tensor memory) = A[m][32] B[n][32]^T (+ D where `more`).
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool more) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(desc), "r"((uint32_t)more)
        : "memory");
}

// ------------------------------------------------------------ cluster
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// Every thread of every CTA of the cluster.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared-memory address `at` in the CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(uint32_t at, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
}

}  // namespace tc
}  // namespace zkv
