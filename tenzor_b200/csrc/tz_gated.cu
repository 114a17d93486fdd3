// tz_gated.cu -- the gated feed-forward block in 16 bits, forward and backward, on tcgen05.
//
//   forward    g = x Wg^T, u = x Wu^T,  h = act(g) * u                    x [T, D], Wg and Wu [F, D], h [T, F]
//   backward   dg = dh * u * act'(g),  du = dh * act(g)                   g and u are computed again
//              dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// One persistent kernel template with four forms (what differs is the operands' layout and the epilogue):
//   FWD  both projections of a tile in one accumulator: its B tile is BN/2 rows of Wg over BN/2 rows of Wu, so
//        one MMA makes the gate and the up columns of the same outputs; the epilogue multiplies them
//   BWD  the same products; the epilogue makes dg and du (16 bits) from them and dh, all in f32 before the
//        one rounding that the tensor core needs for the next products' operands
//   DX   [dg | du] [Wg ; Wu]: one accumulation over both halves; the weights are read MN-major in place
//   DW   dg^T x and du^T x: both operands MN-major in place (the sum runs over tokens); where the tiles do not
//        fill the GPU the tokens are split and the f32 partial sums added in a fixed order by a second kernel
//
// Per CTA (64 + 32 * EPI warps): warp 0 TMA producer, warp 1 allocates TMEM and issues the MMAs, the others
// read the accumulators (two buffers: the epilogue of a tile runs under the next tile's MMAs) and store boxes
// of 32 x 32 outputs through swizzled shared memory and TMA, which clips ragged edges.  TMA fills reads
// outside the operands with zeros, so any T works; D and F are multiples of 8 (16-byte rows).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tz_act.cuh"
#include "tz_gated_rows.cuh"
#include "tz_internal.h"
#include "tz_pair.cuh"

namespace tz {
namespace {

enum { MM_FWD = 0, MM_BWD = 1, MM_DX = 2, MM_DW = 3 };

struct MmParams {
    int m_tiles, n_tiles;  // tiles of 128 * CG rows x BN columns (FWD / BWD: BN / 2 output columns)
    int which;             // DW: 2 (dWg and dWu), else 1
    int splits;            // of the K blocks; > 1: f32 partial sums
    int kblocks;           // K blocks of 64, both halves for DX
    int half;              // DX: K blocks of one half
    int kper;              // K blocks per split
    int ring;              // shared-memory stages in use
    int resident;          // dual forms: the column block's B tiles stay in shared memory (see launch_mm)
    int m_pad;             // rows of one partial sum
    int cols;              // of the output
    int act;
};

template <int CG, int BN, int MODE>
struct MmCfg {
    static constexpr bool kDual = MODE == MM_FWD || MODE == MM_BWD;
    static constexpr bool kAmn = MODE == MM_DW;
    static constexpr bool kBmn = MODE == MM_DX || MODE == MM_DW;
    static constexpr int EPI = kDual ? 16 : 8;
    static constexpr int THREADS = 64 + 32 * EPI;
    static constexpr int BNC = BN / CG;  // B rows (or columns) in one CTA
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int STAGE = A_BYTES + BNC * 128;
    static constexpr int BOX = MODE == MM_FWD ? 2048 : 4096;  // staging of one epilogue warp
    static constexpr int STAGING = EPI * BOX;
    static constexpr int BUDGET = (227 * 1024 - 1024 - 512 - STAGING) / 1024 * 1024;
    static constexpr int STAGES = BUDGET / STAGE > 8 ? 8 : BUDGET / STAGE;
    static constexpr int SMEM = BUDGET + STAGING + 512 + 1024;
    static constexpr int ACCS = BN == 384 ? 1 : 2;  // accumulators in TMEM
    static constexpr int TCOLS = BN == 384 ? 512 : 2 * BN;
    static_assert(!kDual || BN == 256, "16 epilogue warps of 32 output columns");
    static_assert(!kBmn || BNC % 64 == 0, "MN-major B comes in blocks of 64");
    static_assert(BN == 256 || (BN == 384 && kBmn && CG == 2), "384 columns: two MMAs of 256 and 128");
};

// 16 gate / up pairs -> 8 words of 16-bit outputs.
template <int ACT, bool BF>
__device__ __forceinline__ void fwd_math(const uint32_t (&g)[16], const uint32_t (&u)[16], uint32_t* o) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = gated_pair<ACT, BF>(g[2 * j], g[2 * j + 1], u[2 * j], u[2 * j + 1]);
}
template <int ACT, bool BF>
__device__ __forceinline__ void bwd_math(const uint32_t (&g)[16], const uint32_t (&u)[16], const uint32_t* dh, uint32_t* dg, uint32_t* du) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float2 h;
        if constexpr (BF)
            h = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&dh[j]));
        else
            h = __half22float2(*reinterpret_cast<const __half2*>(&dh[j]));
        uint64_t d;
        const uint64_t h2 = tzp::f2_pack(h.x, h.y);
        const uint64_t a = gated_act2<ACT, true>(tzp::f2_pack(__uint_as_float(g[2 * j]), __uint_as_float(g[2 * j + 1])), d);
        const float2 p = tzp::f2_unpack(tzp::f2_mul(tzp::f2_mul(h2, tzp::f2_pack(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1]))), d));
        const float2 q = tzp::f2_unpack(tzp::f2_mul(h2, a));
        dg[j] = tzp::pack16x2<BF>(p.x, p.y);
        du[j] = tzp::pack16x2<BF>(q.x, q.y);
    }
}

// 16-byte units c0 .. c0 + N - 1 of this lane's row of a 32-row box with 64-byte rows and the 64-byte swizzle.
template <int N>
__device__ __forceinline__ void stage64(uint32_t buf, int lane, int c0, const uint32_t* o) {
#pragma unroll
    for (int c = 0; c < N; ++c)
        tzp::st_shared_v4(buf + lane * 64 + (((c0 + c) ^ ((lane >> 1) & 3)) << 4), o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
// 32 rows x 128 bytes into a 4 KB box with the 128-byte swizzle.
__device__ __forceinline__ void stage128(uint32_t buf, int lane, const uint32_t (&v)[32]) {
#pragma unroll
    for (int c = 0; c < 8; ++c)
        tzp::st_shared_v4(buf + lane * 128 + ((c ^ (lane & 7)) << 4), v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}

template <int CG, int BN, int MODE, bool BF, bool PART>
__global__ void __launch_bounds__(MmCfg<CG, BN, MODE>::THREADS, 1)
    gated_mm_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmA1,
                    const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1,
                    const __grid_constant__ CUtensorMap tmO0, const __grid_constant__ CUtensorMap tmO1,
                    const __grid_constant__ CUtensorMap tmDh, const MmParams p, int* status) {
    using C = MmCfg<CG, BN, MODE>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = tzp::smem_u32(smem_raw);
    uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
    uint8_t* staging = smem + C::BUDGET;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint64_t* dhbar = drain + 1;  // one per epilogue warp (BWD)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dhbar + C::EPI);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? tzp::cluster_ctarank() : 0u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tzp::mbar_init(&full[s], 1);
            tzp::mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            tzp::mbar_init(&tfull[a], 1);
            tzp::mbar_init(&tempty[a], C::EPI * CG);
        }
        tzp::mbar_init(drain, 1);
        for (int e = 0; e < C::EPI; ++e) tzp::mbar_init(&dhbar[e], 1);
        *abort_flag = 0;
        tzp::fence_mbar_init();
        tzp::tma_prefetch_desc(&tmA0);
        tzp::tma_prefetch_desc(&tmB0);
    }
    if (warp == 1) tzp::pair_tmem_alloc<CG>(tmem_slot, C::TCOLS);
    tzp::tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) tzp::cluster_sync();  // both CTAs' barriers exist before either signals them
    tzp::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    tzp::pdl_wait();

    // Tile i of this CTA (pair).  Round-robin over the tiles: a group of 8 row blocks walks all column blocks
    // before the next group starts, so that the CTAs running at one time share both operands in L2.  With
    // resident B tiles: a contiguous range of the tiles in column-block order, so that the column block changes
    // rarely.
    const int per = p.m_tiles * p.n_tiles;
    const int num_tiles = per * p.which * p.splits;
    struct Tile {
        int m, n, w, s, kb0, kb1;
    };
    const int me = static_cast<int>(blockIdx.x) / CG, team = static_cast<int>(gridDim.x) / CG;
    const int first = p.resident ? static_cast<int>(static_cast<long long>(num_tiles) * me / team) : 0;
    const int last = p.resident ? static_cast<int>(static_cast<long long>(num_tiles) * (me + 1) / team) : 0;
    auto tile_at = [&](int i, Tile& r) -> bool {
        if (C::kDual && p.resident) {
            const int t = first + i;
            r.n = t / p.m_tiles;
            r.m = t - r.n * p.m_tiles;
            r.w = r.s = r.kb0 = 0;
            r.kb1 = p.kblocks;
            return t < last;
        }
        int t = me + i * team;
        if (t >= num_tiles) return false;
        r.s = t / (per * p.which);
        t -= r.s * per * p.which;
        r.w = t / per;
        t -= r.w * per;
        constexpr int GM = 8;
        const int grp = t / (GM * p.n_tiles);
        const int gm = min(GM, p.m_tiles - grp * GM);
        t -= grp * GM * p.n_tiles;
        r.m = grp * GM + t % gm;
        r.n = t / gm;
        r.kb0 = r.s * p.kper;
        r.kb1 = min(p.kblocks, r.kb0 + p.kper);
        return true;
    };
    auto range_at = [&](int i, int& kb0, int& kb1) -> bool {  // tile_at's K blocks alone, without its divisions
        const int t = C::kDual && p.resident ? first + i : me + i * team;
        kb0 = 0, kb1 = p.kblocks;
        if (p.splits > 1 && t < num_tiles) {
            kb0 = t / (per * p.which) * p.kper;
            kb1 = min(p.kblocks, kb0 + p.kper);
        }
        return t < (C::kDual && p.resident ? last : num_tiles);
    };
    const int ring = p.ring;
    // Shared memory: stage s holds an A tile and a B tile; with resident B tiles a ring of A tiles comes first,
    // then the B tile of every K block.
    const uint32_t sbase = tzp::smem_u32(smem);
    const uint32_t a_step = C::kDual && p.resident ? C::A_BYTES : C::STAGE;
    auto b_addr = [&](int stage, int kb) {
        return C::kDual && p.resident ? sbase + ring * C::A_BYTES + kb * (C::BNC * 128) : sbase + stage * C::STAGE + C::A_BYTES;
    };

    // Column of this CTA's j-th block of 64 of an MN-major B tile.  384 columns are two MMAs: the first takes
    // blocks 0 and 1 of both CTAs (256 columns), the second block 2 (128).
    auto b_col = [&](int n, int j) {
        const int r = static_cast<int>(rank);
        return n * BN + (BN == 384 ? (j < 2 ? 128 * r + 64 * j : 256 + 64 * r) : r * C::BNC + 64 * j);
    };

    if (warp == 0) {
        {
            // ---- TMA producer (the whole warp; one lane issues) ----
            const bool issue = tzp::elect_one();
            int stage = 0;
            uint32_t phase = 0, armed = 0, armed_par = 0;
            bool ok = true;
            Tile q;
            int n_res = -1;  // the column block whose B tiles are resident
            for (int i = 0; ok && tile_at(i, q); ++i) {
                // A B tile is overwritten when its column block is done: the K block that used it last is `kblocks`
                // uses back, and the wait below covers `ring` <= kblocks uses.
                const bool need_b = !(C::kDual && p.resident) || q.n != n_res;
                n_res = q.n;
                const uint32_t bytes = CG * (need_b ? C::STAGE : C::A_BYTES);
                const int m0 = (q.m * CG + static_cast<int>(rank)) * 128;
                for (int kb = q.kb0; kb < q.kb1; ++kb) {
                    if (!tzp::warp_wait(&empty[stage], phase ^ 1u, status, abort_flag)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) {
                        armed |= 1u << stage;
                        armed_par = (armed_par & ~(1u << stage)) | (phase << stage);
                    }
                    const uint32_t bar = CG == 2 ? tzp::mapa(&full[stage], 0) : tzp::smem_u32(&full[stage]);
                    const uint32_t sa = sbase + stage * a_step;
                    const uint32_t sb = b_addr(stage, kb);
                    if (issue) {
                        if (rank == 0) tzp::mbar_arrive_expect_tx(&full[stage], bytes);
                        if constexpr (MODE == MM_DW) {
                            const CUtensorMap* ta = q.w ? &tmA1 : &tmA0;
                            tzp::pair_load_2d<CG>(sa, ta, m0, kb * 64, bar);
                            tzp::pair_load_2d<CG>(sa + 8192, ta, m0 + 64, kb * 64, bar);
#pragma unroll
                            for (int j = 0; j < C::BNC / 64; ++j)
                                tzp::pair_load_2d<CG>(sb + j * 8192, &tmB0, b_col(q.n, j), kb * 64, bar);
                        } else if constexpr (MODE == MM_DX) {
                            const bool up = kb >= p.half;
                            const int k = (up ? kb - p.half : kb) * 64;
                            tzp::pair_load_2d<CG>(sa, up ? &tmA1 : &tmA0, k, m0, bar);
#pragma unroll
                            for (int j = 0; j < C::BNC / 64; ++j)
                                tzp::pair_load_2d<CG>(sb + j * 8192, up ? &tmB1 : &tmB0, b_col(q.n, j), k, bar);
                        } else {
                            tzp::pair_load_2d<CG>(sa, &tmA0, kb * 64, m0, bar);
                            if (!need_b) {
                            } else if constexpr (CG == 2) {
                                tzp::pair_load_2d<CG>(sb, rank ? &tmB1 : &tmB0, kb * 64, q.n * (BN / 2), bar);
                            } else {
                                tzp::pair_load_2d<CG>(sb, &tmB0, kb * 64, q.n * (BN / 2), bar);
                                tzp::pair_load_2d<CG>(sb + (BN / 2) * 128, &tmB1, kb * 64, q.n * (BN / 2), bar);
                            }
                        }
                    }
                    __syncwarp();
                    if (++stage == ring) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // Every copy has landed before the CTA can exit (bounded; the pair's copies all count on the leader).
            for (int s = 0; s < STAGES; ++s)
                if (armed & (1u << s)) tzp::mbar_wait(&full[s], (armed_par >> s) & 1u, status, nullptr);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            // ---- MMA issuer (the whole warp; one lane issues) ----
            const bool issue = tzp::elect_one();
            constexpr uint32_t major = (C::kAmn ? 1u << 15 : 0u) | (C::kBmn ? 1u << 16 : 0u);
            constexpr uint32_t idesc = tzp::make_idesc(1, BF ? 1 : 0, 128 * CG, 256) | major;
            constexpr uint32_t idesc_b = tzp::make_idesc(1, BF ? 1 : 0, 128 * CG, 128) | major;  // columns 256 .. 383
            constexpr uint32_t kAstep = C::kAmn ? 2048u >> 4 : 2u, kBstep = C::kBmn ? 2048u >> 4 : 2u;
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            int kb0, kb1;
            for (int i = 0; ok && range_at(i, kb0, kb1); ++i) {
                if (!tzp::warp_wait(&tempty[acc], acc_phase ^ 1u, status, abort_flag)) break;
                tzp::tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!tzp::warp_wait(&full[stage], phase, status, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tzp::tc_fence_after();
                    const uint32_t sa = sbase + stage * a_step;
                    const uint32_t sb = b_addr(stage, kb);
                    const uint64_t ad = C::kAmn ? tzp::sdesc_mn128(sa, 8192) : tzp::sdesc_k128(sa);
                    const uint64_t bd = C::kBmn ? tzp::sdesc_mn128(sb, 8192) : tzp::sdesc_k128(sb);
                    if (issue) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t more = (kb > kb0 || k > 0) ? 1u : 0u;
                            tzp::pair_mma_f16<CG>(d, ad + kAstep * k, bd + kBstep * k, idesc, more);
                            if constexpr (BN == 384)
                                tzp::pair_mma_f16<CG>(d + 256, ad + kAstep * k, bd + (16384u >> 4) + kBstep * k, idesc_b, more);
                        }
                        tzp::pair_commit<CG>(&empty[stage]);
                    }
                    __syncwarp();
                    if (++stage == ring) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (issue) tzp::pair_commit<CG>(&tfull[acc]);
                __syncwarp();
                if (++acc == C::ACCS) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            // Every MMA issued has completed before TMEM is released.
            if (issue) tzp::pair_commit<CG>(drain);
            __syncwarp();
            tzp::mbar_wait(drain, 0, status, nullptr);
        }
    } else {
        // ---- epilogue: a warp reads TMEM lane quarter (warp % 4) and a slice of the columns: 32 outputs of a
        // dual tile (the gate and the up columns of each), half of the columns otherwise ----
        const int e = warp - 2, q4 = warp & 3, sl = e >> 2;
        const uint32_t box = tzp::smem_u32(staging) + static_cast<uint32_t>(e * C::BOX);
        uint8_t* boxp = staging + e * C::BOX;
        int acc = 0, nb = 0;
        uint32_t acc_phase = 0, dh_phase = 0;
        // BWD: the 32 x 32 box of dh that a tile needs comes by TMA into the first half of the warp's staging; once it
        // is in registers the next tile's is asked for.  dg and du take turns in the second half.
        auto fetch_dh = [&](const Tile& q) {
            tzp::mbar_arrive_expect_tx(&dhbar[e], 2048);
            tzp::tma_load_2d(boxp, &tmDh, q.n * (BN / 2) + sl * 32, (q.m * CG + static_cast<int>(rank)) * 128 + q4 * 32, &dhbar[e]);
        };
        Tile q, next;
        bool more = tile_at(0, next), fetched = false;
        if constexpr (MODE == MM_BWD) {
            fetched = more;
            if (lane == 0 && more) fetch_dh(next);
        }
        for (int i = 1; more; ++i) {
            q = next;
            more = tile_at(i, next);
            if (!more) tzp::pdl_trigger();
            if (!tzp::warp_wait(&tfull[acc], acc_phase, status, abort_flag)) break;
            tzp::tc_fence_after();
            const uint32_t td = tmem_base + (static_cast<uint32_t>(q4 * 32) << 16) + static_cast<uint32_t>(acc * BN);
            const int row0 = (q.m * CG + static_cast<int>(rank)) * 128 + q4 * 32;
            if constexpr (C::kDual) {
                const int cc = sl * 32;
                const int col0 = q.n * (BN / 2) + cc;
                uint32_t dh[16];
                if constexpr (MODE == MM_BWD) {
                    if (!tzp::warp_wait(&dhbar[e], dh_phase, status, abort_flag)) break;
                    dh_phase ^= 1u;
                    fetched = more;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint4 v = ld_shared_v4(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
                        dh[4 * c] = v.x, dh[4 * c + 1] = v.y, dh[4 * c + 2] = v.z, dh[4 * c + 3] = v.w;
                    }
                    __syncwarp();  // every lane has its row
                    if (lane == 0 && more) fetch_dh(next);
                }
                if (lane == 0) tzp::bulk_wait_read<0>();  // the previous tile's last store has read the box
                __syncwarp();
                uint32_t o[16];
#pragma unroll
                for (int c = 0; c < 2; ++c) {  // 16 outputs at a time
                    uint32_t g[16], u[16];
                    tzp::tmem_ld16(td + cc + 16 * c, g);
                    tzp::tmem_ld16(td + BN / 2 + cc + 16 * c, u);
                    tzp::tmem_ld_wait();
                    if (c == 1) {  // the accumulator is in registers: the MMAs may have it back
                        tzp::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (CG == 2)
                                tzp::mbar_arrive_cluster(tzp::mapa(&tempty[acc], 0));
                            else
                                tzp::mbar_arrive(&tempty[acc]);
                        }
                    }
                    if constexpr (MODE == MM_FWD) {
#define TZ_FWD(A) fwd_math<A, BF>(g, u, o + 8 * c)
                        TZ_ACT_SWITCH(p.act, TZ_FWD)
#undef TZ_FWD
                        stage64<2>(box, lane, 2 * c, o + 8 * c);
                    } else {
                        uint32_t o2[8];
#define TZ_BWD(A) bwd_math<A, BF>(g, u, dh + 8 * c, o + 8 * c, o2)
                        TZ_ACT_SWITCH(p.act, TZ_BWD)
#undef TZ_BWD
                        stage64<2>(box + 2048, lane, 2 * c, o2);
                    }
                }
                tzp::fence_proxy_async();
                __syncwarp();
                const bool store = lane == 0 && col0 < p.cols;
                if constexpr (MODE == MM_FWD) {
                    if (store) {
                        tzp::tma_store_2d(&tmO0, boxp, col0, row0);
                        tzp::bulk_commit();
                    }
                } else {
                    if (store) {
                        tzp::tma_store_2d(&tmO1, boxp + 2048, col0, row0);
                        tzp::bulk_commit();
                        tzp::bulk_wait_read<0>();
                    }
                    __syncwarp();
                    stage64<4>(box + 2048, lane, 0, o);
                    tzp::fence_proxy_async();
                    __syncwarp();
                    if (store) {
                        tzp::tma_store_2d(&tmO0, boxp + 2048, col0, row0);
                        tzp::bulk_commit();
                    }
                }
            } else {
                constexpr int CH = BN / 64;
#pragma unroll 1
                for (int c = 0; c < CH; ++c) {
                    const int cc = (sl * CH + c) * 32;
                    const int col0 = q.n * BN + cc;
                    if (col0 >= p.cols) break;
                    uint32_t v[32];
                    tzp::tmem_ld32(td + cc, v);
                    tzp::tmem_ld_wait();
                    if constexpr (PART) {
                        if (lane == 0) tzp::bulk_wait_read<0>();
                        __syncwarp();
                        stage128(box, lane, v);
                        tzp::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            tzp::tma_store_2d(&tmO0, boxp, col0, (q.s * p.which + q.w) * p.m_pad + row0);
                            tzp::bulk_commit();
                        }
                    } else {
                        uint32_t o[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = tzp::pack16x2<BF>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                        if (lane == 0) tzp::bulk_wait_read<1>();
                        __syncwarp();
                        stage64<4>(box + nb * 2048, lane, 0, o);
                        tzp::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            tzp::tma_store_2d(q.w ? &tmO1 : &tmO0, boxp + nb * 2048, col0, row0);
                            tzp::bulk_commit();
                        }
                        nb ^= 1;
                    }
                }
            }
            if constexpr (!C::kDual) {
                tzp::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CG == 2)
                        tzp::mbar_arrive_cluster(tzp::mapa(&tempty[acc], 0));
                    else
                        tzp::mbar_arrive(&tempty[acc]);
                }
            }
            if (++acc == C::ACCS) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        if (lane == 0) {
            tzp::bulk_wait_all();
            if (fetched) tzp::mbar_wait(&dhbar[e], dh_phase, status, nullptr);  // left early: its copy has landed
        }
    }

    if (warp < 2) tzp::pdl_trigger();
    tzp::tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) {
        // The leader's last commit has arrived in CTA 1 too and both CTAs are done: nothing is under way to a
        // CTA that has left.
        if (rank == 1 && threadIdx.x == 32) tzp::mbar_wait(drain, 0, status, nullptr);
        __syncwarp();
        tzp::cluster_sync();
    }
    if (warp == 1) {
        __syncwarp();
        tzp::tc_fence_after();
        tzp::pair_tmem_dealloc<CG>(tmem_base, C::TCOLS);
    }
}

// Sums the partial products [splits][which][m_pad][cols] in order and rounds to 16 bits.
template <bool BF>
__global__ void sum_parts_kernel(const float* part, void* out0, void* out1, int which, int splits, int m_pad, int rows, int cols) {
    const long long n8 = static_cast<long long>(rows) * cols / 8;
    const long long plane = static_cast<long long>(m_pad) * cols;
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < n8 * which; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int w = i >= n8;
        const long long o = (i - (w ? n8 : 0)) * 8;
        float s[8] = {};
        for (int k = 0; k < splits; ++k) {
            const float4* src = reinterpret_cast<const float4*>(part + (static_cast<long long>(k) * which + w) * plane + o);
            const float4 a = __ldcs(src), b = __ldcs(src + 1);
            s[0] += a.x, s[1] += a.y, s[2] += a.z, s[3] += a.w, s[4] += b.x, s[5] += b.y, s[6] += b.z, s[7] += b.w;
        }
        uint4 r = make_uint4(tzp::pack16x2<BF>(s[0], s[1]), tzp::pack16x2<BF>(s[2], s[3]), tzp::pack16x2<BF>(s[4], s[5]), tzp::pack16x2<BF>(s[6], s[7]));
        reinterpret_cast<uint4*>(w ? out1 : out0)[o / 8] = r;
    }
}

// One operand or output of a product: row-major, 16 bits.
struct Mat {
    const void* p;
    int64_t rows, cols, ld;
};

template <bool BF>
int map16(CUtensorMap* m, const Mat& a, int box_cols, int box_rows, CUtensorMapSwizzle swz) {
    return encode_tmap_2d_swz(m, BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, a.p, a.cols, a.rows,
                              a.ld * 2, box_cols, box_rows, swz);
}

template <int CG, int BN, int MODE, bool BF, bool PART>
int launch_mm(tz_ctx_t ctx, const Mat& a0, const Mat& a1, const Mat& b0, const Mat& b1, const Mat& o0, const Mat& o1, const Mat* dh,
              MmParams p, float* part, cudaStream_t s) {
    using C = MmCfg<CG, BN, MODE>;
    auto kern = gated_mm_kernel<CG, BN, MODE, BF, PART>;
    static std::atomic<unsigned> done{0};
    int rc = ensure_smem(kern, C::SMEM, done);
    if (rc) return rc;
    CUtensorMap ma0, ma1, mb0, mb1, mo0, mo1, mdh;
    const auto S128 = CU_TENSOR_MAP_SWIZZLE_128B;
    const int arows = C::kAmn ? 64 : 128, brows = C::kBmn ? 64 : (C::kDual ? BN / 2 : C::BNC);
    if ((rc = map16<BF>(&ma0, a0, 64, arows, S128)) || (rc = map16<BF>(&mb0, b0, 64, brows, S128))) return rc;
    ma1 = ma0, mb1 = mb0;  // an encoding costs about as much as the rest of the launch's arguments
    if (a1.p != a0.p && (rc = map16<BF>(&ma1, a1, 64, arows, S128))) return rc;
    if (b1.p != b0.p && (rc = map16<BF>(&mb1, b1, 64, brows, S128))) return rc;
    if (PART) {
        rc = encode_tmap_2d_swz(&mo0, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, part, o0.cols,
                                static_cast<uint64_t>(p.splits) * p.which * p.m_pad, o0.cols * 4, 32, 32, S128);
        mo1 = mo0;
    } else {
        rc = map16<BF>(&mo0, o0, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
        mo1 = mo0;
        if (!rc && o1.p != o0.p) rc = map16<BF>(&mo1, o1, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    }
    if (rc) return rc;
    mdh = mo0;
    if (dh && (rc = map16<BF>(&mdh, *dh, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B))) return rc;
    const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles * p.which * p.splits;
    const int groups = (ctx->sm_count - ctx->sm_reserve) / CG;
    const int grid = static_cast<int>(tiles < groups ? tiles : groups) * CG;
    TZ_CHECK(grid > 0, TZ_EINVAL, "gated kernels need %d free SMs", CG);
    p.ring = C::STAGES;
    if (C::kDual && tiles > groups && p.kblocks >= 4) {
        // Short sums: the B tiles of a whole column block fit beside a ring of A tiles, and keeping them halves what
        // an SM moves from L2 per tile, which bounds these shapes.  Below 4 K blocks the ring (at most kblocks long)
        // would be too short; above, it has to keep 3 A tiles.
        const int left = (C::BUDGET - p.kblocks * C::BNC * 128) / C::A_BYTES;
        int r = left < p.kblocks ? left : p.kblocks;
        if (r > C::STAGES) r = C::STAGES;
        if (r >= 3) {
            p.resident = 1;
            p.ring = r;
        }
    }
    return launch_cluster(kern, CG, dim3(grid), dim3(C::THREADS), C::SMEM, s, true, ma0, ma1, mb0, mb1, mo0, mo1, mdh, p, ctx->d_status);
}

constexpr int kCG = 2, kBN = 256;
// Tokens up to which the forward pass streams weights (gated_rows_kernel).  At 32 tokens it takes 5.2 / 10.2 /
// 14.5 / 26.8 us at (D, F) = (384, 1536) / (1024, 4096) / (2048, 6144) / (4096, 8192), the tiles of 256 tokens 6.5
// / 10.4 / 16.1 / 29.2; with room for 64 tokens it takes 6.5 / 14.2 / 16.9 / 29.1.
constexpr int kRowsMax = 32;

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

// Tile width and splits of the sum of a DX or DW product, by an estimate in clocks: rounds of tiles over the
// pairs, each K block at the rate the operands arrive at (256 columns: 32 KB per SM, 384: 40 KB), a start and an
// epilogue per round (not hidden with one accumulator), and the partial sums' way out and back.
struct Split {
    int bn, splits;
};
Split pick_split(int sms, int64_t m_tiles, int which, int64_t rows, int64_t cols, int kblocks) {
    const int64_t groups = sms / kCG > 0 ? sms / kCG : 1;
    Split best{256, 1};
    if (kblocks < 1) return best;  // no tokens
    double best_cost = 1e300;
    for (int bn = 256; bn <= 384; bn += 128) {
        const int64_t tiles = m_tiles * which * ceil_div(cols, bn);
        for (int sp = 1; sp <= 16; ++sp) {
            if (sp > 1 && (kblocks / sp < 8 || tiles * sp > groups)) break;
            const int per = ceil_div(kblocks, sp);
            if (ceil_div(kblocks, per) != sp) continue;  // every split has work
            double cost = static_cast<double>(ceil_div(tiles * sp, groups)) * (bn == 256 ? per * 600.0 + 2500.0 : per * 820.0 + 5000.0);
            if (sp > 1) cost += 6000.0 + static_cast<double>(sp) * which * rows * cols * 8.0 / 2500.0;
            if (cost < best_cost) {
                best_cost = cost;
                best = {bn, sp};
            }
        }
    }
    return best;
}

struct BwdPlan {
    size_t dgdu, part_dx, part_dw;  // bytes
    Split dx, dw;
};
BwdPlan plan_bwd(int sms, int64_t T, int64_t D, int64_t F) {
    BwdPlan b{};
    auto a256 = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
    b.dgdu = a256(static_cast<size_t>(T) * F * 2);
    const int mt = ceil_div(T, 128 * kCG), ft = ceil_div(F, 128 * kCG);
    b.dx = pick_split(sms, mt, 1, T, D, 2 * ceil_div(F, 64));
    b.dw = pick_split(sms, ft, 2, F, D, ceil_div(T, 64));
    if (b.dx.splits > 1) b.part_dx = a256(static_cast<size_t>(b.dx.splits) * mt * 128 * kCG * D * 4);
    if (b.dw.splits > 1) b.part_dw = a256(static_cast<size_t>(b.dw.splits) * 2 * ft * 128 * kCG * D * 4);
    return b;
}

template <bool BF>
int sum_parts(tz_ctx_t ctx, const float* part, void* o0, void* o1, int which, int splits, int m_pad, int rows, int cols, cudaStream_t s) {
    const long long n8 = static_cast<long long>(rows) * cols / 8 * which;
    const int blocks = static_cast<int>(n8 / 256 + 1 < ctx->sm_count * 8 ? n8 / 256 + 1 : ctx->sm_count * 8);
    return launch_kernel(sum_parts_kernel<BF>, dim3(blocks), dim3(256), 0, s, false, part, o0, o1, which, splits, m_pad, rows, cols);
}

template <int MODE, bool BF>
int launch_any(tz_ctx_t ctx, const Split& w, const Mat& a0, const Mat& a1, const Mat& b0, const Mat& b1, const Mat& o0, const Mat& o1,
               const MmParams& p, float* part, cudaStream_t s) {
    if (w.bn == 384)
        return p.splits > 1 ? launch_mm<kCG, 384, MODE, BF, true>(ctx, a0, a1, b0, b1, o0, o1, nullptr, p, part, s)
                            : launch_mm<kCG, 384, MODE, BF, false>(ctx, a0, a1, b0, b1, o0, o1, nullptr, p, nullptr, s);
    return p.splits > 1 ? launch_mm<kCG, kBN, MODE, BF, true>(ctx, a0, a1, b0, b1, o0, o1, nullptr, p, part, s)
                        : launch_mm<kCG, kBN, MODE, BF, false>(ctx, a0, a1, b0, b1, o0, o1, nullptr, p, nullptr, s);
}

template <int N, bool BF>
int launch_rows(tz_ctx_t ctx, const Mat& x, const Mat& wg, const Mat& wu, const Mat& h, int act, cudaStream_t s) {
    using C = RowsCfg<N>;
    auto kern = gated_rows_kernel<N, BF>;
    static std::atomic<unsigned> done{0};
    int rc = ensure_smem(kern, C::SMEM, done);
    if (rc) return rc;
    CUtensorMap mx, mg, mu;
    const auto S128 = CU_TENSOR_MAP_SWIZZLE_128B;
    if ((rc = map16<BF>(&mx, x, 64, N, S128)) || (rc = map16<BF>(&mg, wg, 64, 128, S128)) || (rc = map16<BF>(&mu, wu, 64, 128, S128))) return rc;
    RowsParams p{};
    const int tiles = ceil_div(h.cols, 128);
    p.kblocks = ceil_div(x.cols, 64);
    int splits = 1;
    if ((rc = rows_splits<N>(kern, C::THREADS, [](int) { return C::SMEM; }, ctx->sm_count - ctx->sm_reserve, tiles, p.kblocks, C::MAX_SPLIT, &splits))) return rc;
    p.kper = ceil_div(p.kblocks, splits);
    p.t = static_cast<int>(x.rows);
    p.f = static_cast<int>(h.cols);
    p.act = act;
    p.h = const_cast<void*>(h.p);
    return launch_cluster(kern, splits, dim3(splits, tiles), dim3(C::THREADS), C::SMEM, s, true, mx, mg, mu, p, ctx->d_status);
}

template <bool BF>
int forward(tz_ctx_t ctx, const Mat& x, const Mat& wg, const Mat& wu, const Mat& h, int act, cudaStream_t s) {
    if (x.rows <= kRowsMax && h.cols <= 128 * 65535) {  // the grid's second extent
        if (x.rows <= 16) return launch_rows<16, BF>(ctx, x, wg, wu, h, act, s);
        return launch_rows<32, BF>(ctx, x, wg, wu, h, act, s);
    }
    MmParams p{};
    p.m_tiles = ceil_div(x.rows, 128 * kCG);
    p.n_tiles = ceil_div(h.cols, kBN / 2);
    p.which = p.splits = 1;
    p.kblocks = p.kper = ceil_div(x.cols, 64);
    p.cols = static_cast<int>(h.cols);
    p.act = act;
    if (x.rows <= 128 && p.n_tiles > (ctx->sm_count - ctx->sm_reserve) / 2)  // half of a pair's rows would be empty
        return launch_mm<1, kBN, MM_FWD, BF, false>(ctx, x, x, wg, wu, h, h, nullptr, p, nullptr, s);
    return launch_mm<kCG, kBN, MM_FWD, BF, false>(ctx, x, x, wg, wu, h, h, nullptr, p, nullptr, s);
}

template <bool BF>
int backward(tz_ctx_t ctx, const Mat& x, const Mat& wg, const Mat& wu, const Mat& dh, const Mat& dx, const Mat& dwg, const Mat& dwu,
             int act, char* ws, cudaStream_t s) {
    const int64_t T = x.rows, D = x.cols, F = dh.cols;
    const BwdPlan b = plan_bwd(ctx->sm_count - ctx->sm_reserve, T, D, F);
    const Mat dg{ws, T, F, F}, du{ws + b.dgdu, T, F, F};
    float* part_dx = reinterpret_cast<float*>(ws + 2 * b.dgdu);
    float* part_dw = reinterpret_cast<float*>(ws + 2 * b.dgdu + b.part_dx);
    MmParams p{};
    p.m_tiles = ceil_div(T, 128 * kCG);
    p.n_tiles = ceil_div(F, kBN / 2);
    p.which = p.splits = 1;
    p.kblocks = p.kper = ceil_div(D, 64);
    p.cols = static_cast<int>(F);
    p.act = act;
    int rc = launch_mm<kCG, kBN, MM_BWD, BF, false>(ctx, x, x, wg, wu, dg, du, &dh, p, nullptr, s);
    if (rc) return rc;

    MmParams q{};
    q.m_tiles = ceil_div(T, 128 * kCG);
    q.n_tiles = ceil_div(D, b.dx.bn);
    q.which = 1;
    q.splits = b.dx.splits;
    q.half = ceil_div(F, 64);
    q.kblocks = 2 * q.half;
    q.kper = ceil_div(q.kblocks, q.splits);
    q.m_pad = q.m_tiles * 128 * kCG;
    q.cols = static_cast<int>(D);
    rc = launch_any<MM_DX, BF>(ctx, b.dx, dg, du, wg, wu, dx, dx, q, part_dx, s);
    if (!rc && q.splits > 1)
        rc = sum_parts<BF>(ctx, part_dx, const_cast<void*>(dx.p), nullptr, 1, q.splits, q.m_pad, static_cast<int>(T), q.cols, s);
    if (rc) return rc;

    MmParams r{};
    r.m_tiles = ceil_div(F, 128 * kCG);
    r.n_tiles = ceil_div(D, b.dw.bn);
    r.which = 2;
    r.splits = b.dw.splits;
    r.kblocks = ceil_div(T, 64);
    r.kper = ceil_div(r.kblocks, r.splits);
    r.m_pad = r.m_tiles * 128 * kCG;
    r.cols = static_cast<int>(D);
    rc = launch_any<MM_DW, BF>(ctx, b.dw, dg, du, x, x, dwg, dwu, r, part_dw, s);
    if (!rc && r.splits > 1)
        rc = sum_parts<BF>(ctx, part_dw, const_cast<void*>(dwg.p), const_cast<void*>(dwu.p), 2, r.splits, r.m_pad, static_cast<int>(F), r.cols, s);
    return rc;
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_shape(const char* fn, int64_t T, int D, int F, int dtype, int act) {
    TZ_CHECK(dtype == TZ_PREC_F16 || dtype == TZ_PREC_BF16, TZ_EINVAL, "%s: dtype %d is neither f16 nor bf16", fn, dtype);
    TZ_CHECK(gated_act_ok(act), TZ_EINVAL, "%s: activation %d is not silu, gelu, gelu_erf, relu or sigmoid", fn, act);
    TZ_CHECK(T >= 0 && T <= (1 << 30) && D > 0 && F > 0 && D <= (1 << 24) && F <= (1 << 24), TZ_EINVAL, "%s: bad sizes T=%lld D=%d F=%d", fn,
             static_cast<long long>(T), D, F);
    TZ_CHECK(D % 8 == 0 && F % 8 == 0, TZ_EINVAL, "%s: D and F must be multiples of 8 (D=%d F=%d)", fn, D, F);
    return TZ_OK;
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

int tz_gated_linear(tz_ctx_t ctx, const void* x, int64_t ldx, const void* w_gate, const void* w_up, void* h, int64_t t, int d, int f,
                    int act, int dtype, tz_stream_t stream) {
    TZ_CHECK(ctx, TZ_EINVAL, "tz_gated_linear: null context");
    int rc = check_shape("tz_gated_linear", t, d, f, dtype, act);
    if (rc) return rc;
    if (t == 0) return TZ_OK;
    TZ_CHECK(x && w_gate && w_up && h, TZ_EINVAL, "tz_gated_linear: null pointer");
    TZ_CHECK(ldx >= d && ldx % 8 == 0, TZ_EINVAL, "tz_gated_linear: row stride %lld of x (at least D, a multiple of 8)", static_cast<long long>(ldx));
    TZ_CHECK(al16(x) && al16(w_gate) && al16(w_up) && al16(h), TZ_EINVAL, "tz_gated_linear: pointers must be 16-byte aligned");
    cudaStream_t s = pick_stream(ctx, stream);
    const Mat mx{x, t, d, ldx}, mg{w_gate, f, d, d}, mu{w_up, f, d, d}, mh{h, t, f, f};
    return dtype == TZ_PREC_BF16 ? forward<true>(ctx, mx, mg, mu, mh, act, s) : forward<false>(ctx, mx, mg, mu, mh, act, s);
}

int tz_gated_linear_backward_workspace(int sms, int64_t t, int d, int f, size_t* bytes) {
    TZ_CHECK(sms > 0 && bytes, TZ_EINVAL, "tz_gated_linear_backward_workspace: bad argument");
    int rc = check_shape("tz_gated_linear_backward_workspace", t, d, f, TZ_PREC_F16, TZ_OP_SILU);
    if (rc) return rc;
    const BwdPlan b = plan_bwd(sms, t, d, f);
    *bytes = 2 * b.dgdu + b.part_dx + b.part_dw;
    return TZ_OK;
}

int tz_gated_linear_backward(tz_ctx_t ctx, const void* x, int64_t ldx, const void* w_gate, const void* w_up, const void* dh, int64_t lddh,
                             void* dx, void* dw_gate, void* dw_up, void* workspace, size_t workspace_bytes, int64_t t, int d, int f,
                             int act, int dtype, tz_stream_t stream) {
    TZ_CHECK(ctx, TZ_EINVAL, "tz_gated_linear_backward: null context");
    int rc = check_shape("tz_gated_linear_backward", t, d, f, dtype, act);
    if (rc) return rc;
    TZ_CHECK(w_gate && w_up && dw_gate && dw_up && (t == 0 || (x && dh && dx && workspace)), TZ_EINVAL, "tz_gated_linear_backward: null pointer");
    cudaStream_t s = pick_stream(ctx, stream);
    if (t == 0) {  // an empty sum
        TZ_CUDA(cudaMemsetAsync(dw_gate, 0, static_cast<size_t>(d) * f * 2, s));
        TZ_CUDA(cudaMemsetAsync(dw_up, 0, static_cast<size_t>(d) * f * 2, s));
        return TZ_OK;
    }
    TZ_CHECK(ldx >= d && ldx % 8 == 0 && lddh >= f && lddh % 8 == 0, TZ_EINVAL,
             "tz_gated_linear_backward: row strides %lld of x and %lld of dh (at least the width, multiples of 8)", static_cast<long long>(ldx),
             static_cast<long long>(lddh));
    TZ_CHECK(al16(x) && al16(w_gate) && al16(w_up) && al16(dh) && al16(dx) && al16(dw_gate) && al16(dw_up) && al16(workspace), TZ_EINVAL,
             "tz_gated_linear_backward: pointers must be 16-byte aligned");
    size_t need = 0;
    if ((rc = tz_gated_linear_backward_workspace(ctx->sm_count - ctx->sm_reserve, t, d, f, &need))) return rc;
    TZ_CHECK(workspace_bytes >= need, TZ_EINVAL, "tz_gated_linear_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const Mat mx{x, t, d, ldx}, mg{w_gate, f, d, d}, mu{w_up, f, d, d}, mdh{dh, t, f, lddh}, mdx{dx, t, d, d}, mwg{dw_gate, f, d, d},
        mwu{dw_up, f, d, d};
    char* ws = static_cast<char*>(workspace);
    return dtype == TZ_PREC_BF16 ? backward<true>(ctx, mx, mg, mu, mdh, mdx, mwg, mwu, act, ws, s)
                                 : backward<false>(ctx, mx, mg, mu, mdh, mdx, mwg, mwu, act, ws, s);
}

}  // extern "C"
