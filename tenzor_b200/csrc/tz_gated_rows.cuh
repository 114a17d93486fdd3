// tz_gated_rows.cuh -- the gated block for few tokens (serving, one token at a time): bound by reading the two
// weight matrices once.  GRAD is the backward pass's first kernel for few tokens: dg and du from the same products.
//
// The tensor core's roles are swapped: 128 rows of Wg and of Wu are the two A tiles (M = 128 output features)
// and up to 32 tokens the B tile (N), so no lane works on padding that costs bandwidth.  The K blocks of a
// feature tile are split over the CTAs of a cluster (up to 8), enough to give every SM a stream of weights;
// the f32 partial sums of the other CTAs go to the first one's shared memory and are added there in rank
// order.  Against the 256 x 256 tiles of the large kernel, which give a CTA pair 128 features and leave most
// pairs without work at these sizes, each SM keeps 6 x 32 KB of weights in flight.
//
// Measured (bf16, one token, weights from DRAM): D = 4096, F = 16384 43.5 us, 6.2 TB/s, 94 % of the measured copy
// rate; D = 4096, F = 8192 24.7 us; D = 2048, F = 6144 12.4 us, of which about 4 us are the launch, the first
// loads' latency and the join.
#pragma once
#include "tz_act.cuh"
#include "tz_internal.h"
#include "tz_pair.cuh"

namespace tz {

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// A packed 16-bit pair as f32.
template <bool BF>
__device__ __forceinline__ float2 widen2(uint32_t w) {
    if constexpr (BF)
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    else
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

struct RowsParams {
    int kblocks, kper;  // K blocks of 64, and of one cluster rank
    int tile0;          // the launch's first feature tile
    int t, f, act;
    void* h;         // GRAD: dg
    void* du;        // GRAD
    const void* dh;  // GRAD: [t, f], row stride lddh
    long long lddh;
};

template <int N>
struct RowsCfg {
    static constexpr int THREADS = 64 + 128;
    static constexpr int STAGE = 2 * 16384 + N * 128;
    static constexpr int STAGES = 6 * STAGE + 2048 <= 227 * 1024 ? 6 : 5;
    static constexpr int SMEM = STAGES * STAGE + 512 + 1024;
    static constexpr int TCOLS = 2 * N < 32 ? 32 : 2 * N;
    static constexpr int PART = 128 * 2 * N * 4;  // one rank's partial sums
    static constexpr int MAX_SPLIT = 1 + STAGES * STAGE / PART;
};

template <int N, bool BF, bool GRAD>
__global__ void __launch_bounds__(RowsCfg<N>::THREADS, 1)
    gated_rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmG, const __grid_constant__ CUtensorMap tmU,
                      const RowsParams p, int* status) {
    using C = RowsCfg<N>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (tzp::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE);
    uint64_t* empty = full + STAGES;
    uint64_t* done = empty + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(tzp::cluster_ctarank());
    const int f0 = (p.tile0 + static_cast<int>(blockIdx.y)) * 128;
    const int kb0 = rank * p.kper, kb1 = min(p.kblocks, kb0 + p.kper);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tzp::mbar_init(&full[s], 1);
            tzp::mbar_init(&empty[s], 1);
        }
        tzp::mbar_init(done, 1);
        *abort_flag = 0;
        tzp::fence_mbar_init();
        tzp::tma_prefetch_desc(&tmX);
        tzp::tma_prefetch_desc(&tmG);
        tzp::tma_prefetch_desc(&tmU);
    }
    if (warp == 1) {
        tzp::tmem_alloc(tmem_slot, C::TCOLS);
        tzp::tmem_relinquish();
    }
    tzp::tc_fence_before();
    __syncthreads();
    tzp::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    tzp::pdl_wait();

    if (warp == 0) {
        {  // the whole warp; one lane issues
            const bool issue = tzp::elect_one();
            uint32_t armed = 0, armed_par = 0;
            for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
                const int s = i % STAGES;
                const uint32_t phase = (i / STAGES) & 1;
                if (!tzp::warp_wait(&empty[s], phase ^ 1u, status, abort_flag)) break;
                uint8_t* a = smem + s * C::STAGE;
                armed |= 1u << s;
                armed_par = (armed_par & ~(1u << s)) | (phase << s);
                if (issue) {
                    tzp::mbar_arrive_expect_tx(&full[s], C::STAGE);
                    tzp::tma_load_2d(a, &tmG, kb * 64, f0, &full[s]);
                    tzp::tma_load_2d(a + 16384, &tmU, kb * 64, f0, &full[s]);
                    tzp::tma_load_2d(a + 32768, &tmX, kb * 64, 0, &full[s]);
                }
                __syncwarp();
            }
            for (int s = 0; s < STAGES; ++s)  // every copy has landed before the stages are used again (bounded)
                if (armed & (1u << s)) tzp::mbar_wait(&full[s], (armed_par >> s) & 1u, status, nullptr);
        }
    } else if (warp == 1) {
        {  // the whole warp; one lane issues
            const bool issue = tzp::elect_one();
            constexpr uint32_t idesc = tzp::make_idesc(1, BF ? 1 : 0, 128, N);
            for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
                const int s = i % STAGES;
                if (!tzp::warp_wait(&full[s], (i / STAGES) & 1, status, abort_flag)) break;
                tzp::tc_fence_after();
                const uint32_t a = tzp::smem_u32(smem + s * C::STAGE);
                const uint64_t gd = tzp::sdesc_k128(a), ud = tzp::sdesc_k128(a + 16384), xd = tzp::sdesc_k128(a + 32768);
                if (issue) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        tzp::umma<0>(tmem_base, gd + 2u * k, xd + 2u * k, idesc, (i | k) != 0 ? 1u : 0u);
                        tzp::umma<0>(tmem_base + N, ud + 2u * k, xd + 2u * k, idesc, (i | k) != 0 ? 1u : 0u);
                    }
                    tzp::umma_commit(&empty[s]);
                }
                __syncwarp();
            }
            if (issue) tzp::umma_commit(done);
            __syncwarp();
            tzp::mbar_wait(done, 0, status, nullptr);
        }
    }
    // All products of this CTA are in its TMEM and its stages are free; then the same of every CTA.
    tzp::tc_fence_before();
    __syncthreads();
    const bool split = p.kper < p.kblocks;
    if (split) tzp::cluster_sync();
    tzp::tc_fence_after();

    const int q4 = warp & 3, row = q4 * 32 + lane;  // output feature f0 + row
    float* part = reinterpret_cast<float*>(smem);   // [rank - 1][2 N][128]
    const uint32_t td = tmem_base + (static_cast<uint32_t>(q4 * 32) << 16);
    if (rank > 0 && warp >= 2) {
        const uint32_t dst = tzp::mapa(part + (rank - 1) * 2 * N * 128 + row, 0);
#pragma unroll 1
        for (int c = 0; c < 2 * N; c += 16) {
            uint32_t v[16];
            tzp::tmem_ld16(td + c, v);
            tzp::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) st_cluster_f32(dst + (c + j) * 512, __uint_as_float(v[j]));
        }
    }
    if (split) tzp::cluster_sync();
    if (rank == 0 && warp >= 2) {
        const int ranks = (p.kblocks + p.kper - 1) / p.kper;
        uint16_t* out = reinterpret_cast<uint16_t*>(p.h) + f0 + row;
        uint16_t* out2 = reinterpret_cast<uint16_t*>(p.du) + f0 + row;
#pragma unroll 1
        for (int c = 0; c < N; c += 16) {
            if (c >= p.t) break;
            uint32_t g[16], u[16];
            tzp::tmem_ld16(td + c, g);
            tzp::tmem_ld16(td + N + c, u);
            tzp::tmem_ld_wait();
            for (int r = 1; r < ranks; ++r) {
                const float* src = part + (r - 1) * 2 * N * 128 + row;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    g[j] = __float_as_uint(__uint_as_float(g[j]) + src[(c + j) * 128]);
                    u[j] = __float_as_uint(__uint_as_float(u[j]) + src[(N + c + j) * 128]);
                }
            }
            uint32_t o[8], o2[8];
            if constexpr (GRAD) {
                const uint16_t* src = reinterpret_cast<const uint16_t*>(p.dh) + f0 + row;
                uint32_t dh[8];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint32_t v = f0 + row < p.f && c + j < p.t ? __ldg(src + (c + j) * p.lddh) : 0;
                    dh[j / 2] = j & 1 ? dh[j / 2] | v << 16 : v;
                }
#define TZ_ROWS(A) \
    for (int j = 0; j < 8; ++j) gated_pair_grad<A, BF>(g[2 * j], g[2 * j + 1], u[2 * j], u[2 * j + 1], widen2<BF>(dh[j]), o[j], o2[j])
                TZ_ACT_SWITCH(p.act, _Pragma("unroll") TZ_ROWS)
#undef TZ_ROWS
            } else {
#define TZ_ROWS(A) \
    for (int j = 0; j < 8; ++j) o[j] = gated_pair<A, BF>(g[2 * j], g[2 * j + 1], u[2 * j], u[2 * j + 1])
                TZ_ACT_SWITCH(p.act, _Pragma("unroll") TZ_ROWS)
#undef TZ_ROWS
            }
            if (f0 + row < p.f) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (c + j >= p.t) break;
                    const long long at = static_cast<long long>(c + j) * p.f;
                    out[at] = static_cast<uint16_t>(o[j / 2] >> (16 * (j & 1)));
                    if constexpr (GRAD) out2[at] = static_cast<uint16_t>(o2[j / 2] >> (16 * (j & 1)));
                }
            }
        }
    }
    tzp::pdl_trigger();
    tzp::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tzp::tc_fence_after();
        tzp::tmem_dealloc(tmem_base, C::TCOLS);
    }
}

// K splits of a feature tile: the most (up to 8, each with at least 4 K blocks) with which the clusters of all
// tiles still run at one time.  How many clusters of a size and shared memory (`smem` of the K blocks of one rank)
// fit is asked of the runtime once: their CTAs have to lie in one GPC, so 148 SMs hold fewer than 148 / size of
// them (48 tiles as clusters of 3 took two waves, 18.5 us, where clusters of 2 take one, 12.4 us).  TAG: one per
// kernel.
template <int TAG, typename K, typename Smem>
int rows_splits(K kern, int threads, Smem smem, int max_ctas, int tiles, int kblocks, int most, int* out) {
    static std::atomic<int> fit[16][9][33];  // by device, size and K blocks of a rank (32: or more); 0 = not asked
    int dev = 0;
    TZ_CUDA(cudaGetDevice(&dev));
    *out = 1;
    for (int s = most < 8 ? most : 8; s > 1; --s) {
        if (kblocks < 4 * s || static_cast<int64_t>(tiles) * s > max_ctas) continue;
        const int per = (kblocks + s - 1) / s;
        if ((kblocks + per - 1) / per != s) continue;  // every rank has work
        if (smem(per < 32 ? per : 32) > 227 * 1024) continue;
        std::atomic<int>& slot = fit[dev & 15][s][per < 32 ? per : 32];
        int n = slot.load(std::memory_order_relaxed);
        if (n == 0) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(s);
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem(per < 32 ? per : 32);
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = s;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            TZ_CUDA(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
            n = n > 0 ? n : -1;
            slot.store(n, std::memory_order_relaxed);
        }
        if (tiles <= n) {
            *out = s;
            return TZ_OK;
        }
    }
    return TZ_OK;
}

// The launches of a few-row kernel's feature tiles, launch(first tile, tiles, pdl): one for all of them, or, where SMs
// are reserved and the tiles are more than the CTAs that the others hold at a time, one for as many tiles as there are
// SMs left, and so on, each after the one before is done.  (rows_splits gives no cluster to tiles that do not fit.)
template <typename Launch>
int rows_launches(tz_ctx_t ctx, int tiles, int splits, Launch launch) {
    const int at_once = (ctx->sm_count - ctx->sm_reserve) / splits;
    const int step = ctx->sm_reserve > 0 && tiles > at_once ? at_once : tiles;
    for (int t = 0; t < tiles; t += step) {
        const int rc = launch(t, tiles - t < step ? tiles - t : step, t == 0);
        if (rc) return rc;
    }
    return TZ_OK;
}

}  // namespace tz
