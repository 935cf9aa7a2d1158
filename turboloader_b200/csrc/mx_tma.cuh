// mbarriers, tensor-map copies and tensor-core instructions used by the microscaled products.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace tlb {

constexpr int kSms = 148;
constexpr unsigned long long kGiveUpNs = 4000000000ull;  // a wait that lasts this long is given up

__device__ __forceinline__ unsigned smem_u32(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ bool elect_one() {  // one lane of a converged warp
    unsigned one;
    asm volatile("{ .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Counts bytes as landed that no copy will bring.
__device__ __forceinline__ void mbar_complete_tx(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile(
        "{ .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for a phase, a whole warp together; false (in all lanes) when the wait was given up, here or by another warp of
// the CTA.  A CTA that gave up ends in order: every role leaves its loop, what it has not summed is written as NaN,
// copies in flight are waited for (Pair), TMEM is freed.
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, volatile int* gave_up) {
    if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
    const unsigned long long began = now_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
        if (now_ns() - began > kGiveUpNs) *gave_up = 1;
        if (__any_sync(0xffffffffu, *gave_up)) return false;
    }
}

// Two CTAs work as a pair (a cluster of 2): rank 0 leads, issues the tensor-core work of both and owns the
// barriers that copies and epilogues of either arrive on.
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned at_rank(unsigned addr, unsigned rank) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ unsigned at_leader(unsigned addr) { return at_rank(addr, 0); }
__device__ __forceinline__ void store_at(unsigned cluster_addr, unsigned v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_at(unsigned cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// What the CTAs of a pair tell each other for their end, in the shared memory of both (the counts in the leader's).
struct Pair {
    unsigned gave_up;         // one of them did
    unsigned started[2][2];   // copies that each rank started: into the ring, and of A into its slots
};
// Waits for the copies that either rank of the pair started and that nothing has waited for: the last ones round a
// ring of barriers that count a share of each rank.  A copy that one rank started and the other did not is made whole:
// the leader's arrival, or the missing share.  A warp of the leader, after the pair has met.
__device__ __forceinline__ void wait_for_copies(unsigned bars, unsigned ring, unsigned mine, unsigned other, unsigned share) {
    int none = 0;
    const bool one = elect_one();
    const unsigned most = mine > other ? mine : other;
    for (unsigned j = most > ring ? most - ring : 0; j < most; ++j) {
        const unsigned bar = bars + 8 * (j % ring);
        if (one && j >= mine) mbar_arrive_tx(bar, share);
        else if (one && j >= other) mbar_complete_tx(bar, share);
        __syncwarp();
        mbar_wait(bar, (j / ring) & 1, &none);
    }
}
// A box of a 2-D map into this CTA's shared memory, counted on a barrier of this CTA or of the leader.
__device__ __forceinline__ void tma_load_2d(unsigned dst, const CUtensorMap* map, int x, int y, unsigned bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Where stored lines stand in L2's order of eviction: first (large results, which L2 cannot keep anyway) or as usual.
__device__ __forceinline__ unsigned long long store_policy(bool passing) {
    unsigned long long p;
    if (passing) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, unsigned src, unsigned long long policy) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%1, %2}], [%3], %4;" ::"l"(map), "r"(x), "r"(y),
                 "r"(src), "l"(policy)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// All lanes of one warp in each CTA of the pair; the base address lands in shared memory at `dst`.
__device__ __forceinline__ void tmem_alloc(unsigned dst, unsigned columns) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(unsigned base, unsigned columns) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}

// Arrives on `bar` of both CTAs when the tensor-core work issued so far by this thread is done.
__device__ __forceinline__ void tc_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<unsigned short>(3))
                 : "memory");
}

// Programmatic launches: the next kernel may start (its own wait still waits for this one's end) / wait for
// the kernel before.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 16 consecutive fp32 columns of the 32 TMEM lanes that this warp may read.
__device__ __forceinline__ void tmem_load16(unsigned addr, unsigned v[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor: bits 0-13 address / 16, 16-29 leading offset / 16, 32-45 stride offset / 16,
// 46 descriptor version 1, 61-63 layout (0: none, 2: 128-byte swizzle).
__device__ __forceinline__ unsigned long long smem_desc(unsigned addr, unsigned leading, unsigned stride, unsigned layout) {
    return static_cast<unsigned long long>((addr & 0x3ffffu) >> 4) | (static_cast<unsigned long long>(leading >> 4) << 16) |
           (static_cast<unsigned long long>(stride >> 4) << 32) | (1ull << 46) | (static_cast<unsigned long long>(layout) << 61);
}

}  // namespace tlb
