// tz_pair.cuh -- what the two-SM (CTA pair) tensor-core kernels share on top of tz_ptx.cuh: TMA loads,
// barriers, tcgen05 allocation, MMA and commit for cta_group::1 and cta_group::2, and the launch with a
// cluster size.
//
// A pair is a cluster of two CTAs whose tensor cores work on one tile: each CTA holds its own 128 rows of A
// and half of B in its own shared memory at the same offsets, and its own 128 rows of the accumulator in its
// own TMEM at the same columns.  CTA 0 (the leader) issues the MMAs for both.  The copies of both CTAs
// complete on the leader's barrier; the commits arrive on both CTAs' barriers.  No TMA multicast is used.
#pragma once
#include <atomic>

#include "tz_internal.h"
#include "tz_ptx.cuh"

namespace tzp {

// One lane of a converged warp (always the same one).  The MMA issuers run their loops with the whole warp and
// issue under this predicate: addresses and descriptors then stay in uniform registers, where a branch on the
// lane number moves each operand of each instruction there one by one.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Address of the same shared-memory variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t mapa(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival on the barrier at a cluster address.  Relaxed: it releases TMEM that this thread has read, which
// tcgen05.wait::ld and tcgen05.fence::before_thread_sync order; a release at cluster scope would hold the warp
// until its earlier memory operations are done (1500 of the 5000 clocks of a gated tile's epilogue).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// A whole warp's bounded wait, with one answer for all lanes (a wait that ran out in one lane must not split the
// warp).  What the waiting side then reads was written by TMA or by tcgen05, ordered by the barrier's byte count and
// the tcgen05 fences, so the plain CTA-scope form does for the barriers that the other CTA of a pair signals too.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, volatile int* abort) {
    if (__all_sync(0xFFFFFFFFu, mbar_try_wait(smem_u32(bar), parity))) return true;
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, status, abort));
}

// 2-D tiled load into this CTA's shared memory, its bytes counted on the barrier at cluster address `bar`
// (the leader's, for a pair).
template <int CG>
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* m, int32_t x, int32_t y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(bar)
            : "memory");
}

template <int CG>
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* slot, uint32_t ncols) {
    if constexpr (CG == 1) {
        tmem_alloc(slot, ncols);
        tmem_relinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(ncols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    if constexpr (CG == 1)
        tmem_dealloc(taddr, ncols);
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Arrives on `bar` (of both CTAs, for a pair) once the tcgen05 operations issued so far have completed.
template <int CG>
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    if constexpr (CG == 1)
        umma_commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"(static_cast<uint16_t>(3))
            : "memory");
}
// D (+)= A B^T for 16-bit operands, f32 accumulator.
template <int CG>
__device__ __forceinline__ void pair_mma_f16(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        umma<0>(d, ad, bd, idesc, accumulate);
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
            : "memory");
}

// Descriptor of an MN-major 16-bit operand tile: blocks of 64 MN elements (128-byte rows, one per k,
// 128-byte swizzle), `lbo` bytes apart; 8-row k groups 1024 bytes apart (SBO).
__device__ __forceinline__ uint64_t sdesc_mn128(uint32_t smem_addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(lbo >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

}  // namespace tzp

namespace tz {

// launch_kernel with a cluster of `cg` CTAs (grid.x a multiple of cg).
//
// Programmatic launches and progress.  A dependent grid is scheduled once every CTA of the grid before it has issued
// launch_dependents or ended, so all clusters of that grid are placed by then.  The cluster kernels issue it at a CTA's
// last tile (the few-row kernels at its end), long after their TMEM is allocated, so that no dependent holds threads,
// shared memory or TMEM for the length of a grid, or takes TMEM that the awaited grid has still to ask for; the small
// kernels around them (quantisers, partial sums) are launched without the attribute.  Waits on an mbarrier are bounded.
// The three others end because
//   griddepcontrol.wait  waits for grids earlier in the stream, whose CTAs have all started (above) and which end by
//                        the same reasons;
//   tcgen05.alloc        waits for columns of CTAs on the same SM.  A CTA of a tile kernel or of the 16-bit few-row
//                        kernel (204 KB of shared memory or more) leaves no room for another that uses TMEM; 4-bit
//                        few-row CTAs (73 KB or more: three to an SM) take 128 of the 512 columns each, so they never
//                        wait for one another; and the other kernels that use TMEM have no clusters, so a CTA of
//                        theirs that holds columns ends without any CTA that waits for them;
//   barrier.cluster      the CTAs of a cluster are placed together, and each arrives after waits of the kinds above.
template <typename... KArgs, typename... Args>
int launch_cluster(void (*kern)(KArgs...), int cg, dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl,
                   Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cg;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
    if (e != cudaSuccess) return cuda_fail(e, "cudaLaunchKernelEx");
    return TZ_OK;
}

// Raises a kernel's dynamic shared-memory limit once per device.
template <typename K>
int ensure_smem(K kern, int bytes, std::atomic<unsigned>& done) {
    int dev = 0;
    TZ_CUDA(cudaGetDevice(&dev));
    const unsigned bit = 1u << (dev & 31);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        TZ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(bit, std::memory_order_release);
    }
    return TZ_OK;
}

}  // namespace tz
