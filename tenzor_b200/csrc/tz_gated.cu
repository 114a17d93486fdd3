// tz_gated.cu -- the gated feed-forward block in 16 bits, forward and backward, on tcgen05.
//
//   forward    g = x Wg^T, u = x Wu^T,  h = act(g) * u                    x [T, D], Wg and Wu [F, D], h [T, F]
//   backward   dg = dh * u * act'(g),  du = dh * act(g)                   g and u are computed again
//              dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// One persistent kernel template with three forms (what differs is the operands' layout and the epilogue):
//   FWD  both projections of a tile in one accumulator: its B tile is BN/2 rows of Wg over BN/2 rows of Wu, so
//        one MMA makes the gate and the up columns of the same outputs; the epilogue multiplies them
//   BWD  the same products; the epilogue makes dg and du (16 bits) from them and dh, all in f32 before the
//        one rounding that the tensor core needs for the next products' operands
//   GRAD dx and both weights' gradients in one launch (the two kinds of tiles fill each other's last round):
//        dx = [dg | du] [Wg ; Wu] is one accumulation over both halves, the weights read MN-major in place;
//        dWg = dg^T x and dWu = du^T x read both operands MN-major in place (the sum runs over tokens).
//        Where the tiles do not fill the SMs in use their sums are split and the f32 partial sums added
//        in a fixed order by a second kernel
//
// Per CTA (64 + 32 * EPI threads): warp 0 TMA producer, warp 1 allocates TMEM and issues the MMAs, the others
// read the accumulators (two buffers: the epilogue of a tile runs under the next tile's MMAs) and store boxes
// of 32 x 32 outputs through swizzled shared memory and TMA, which clips ragged edges.  TMA fills reads
// outside the operands with zeros, so any T works; D and F are multiples of 8 (16-byte rows).
//
// Bounds and measurements (B200; "alone": one launch with idle clocks before it, "in a loop": under the board's power
// cap, which holds the large shapes at 1.1 to 1.5 GHz):
//   T 8192, D 4096, F 8192, bf16   FWD 680 us alone (1.62 PFLOP/s, tensor pipe 98.5 % active), 0.80 ms in a loop;
//                                  BWD 0.70 ms and GRAD 1.51 ms alone (98.7 %), 2.4 to 2.6 ms together in a loop.
//                                  Single CTAs (128 x 256 tiles, cta_group::1) took 0.97 and 2.97 ms in a loop: a pair
//                                  reads each B tile once for 256 rows.
//   T 18106, D 384, F 1536         FWD 36 us alone; a call 33 us in a burst of 21, 42 us sustained at 1.3 GHz (power
//                                  cap).  Six K blocks a tile, so the operand feed from L2 and the epilogue
//                                  (special-function unit 52 %) come close to the MMAs (73 %).  8 epilogue warps took 53 us alone, B tiles loaded for every tile
//                                  48 us in a loop.  BWD 49 us (writes dg and du, 111 MB), GRAD 65 us, sums 8 us.
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

enum { MM_FWD = 0, MM_BWD = 1, MM_GRAD = 2 };

// One product's tiles: m_tiles row blocks of 128 * CG x n_tiles column blocks (FWD / BWD: of BN / 2 outputs).
struct Grid {
    int m_tiles, n_tiles;
    int which;    // products of this shape: 2 for dWg and dWu, else 1
    int splits;   // of the K blocks; > 1: f32 partial sums
    int kblocks;  // K blocks of 64
    int kper;     // K blocks per split
    int m_pad;    // rows of one partial sum
};

struct MmParams {
    Grid g[2];    // GRAD: dx, then the weights' gradients; else g[0] alone
    int ring;     // shared-memory stages in use
    int resident; // dual forms: the column block's B tiles stay in shared memory (see launch_mm)
    int half;     // GRAD: K blocks of one half of dx's sum
    int cols;     // of the output
    int act;
};

// Tensor maps: A (FWD / BWD: x; GRAD: dg and du as dx's operand, then as the weights' gradients'), B (Wg and Wu; GRAD:
// x too), the outputs (h; dg and du; dx, dWg and dWu or their partial sums), and dh.
struct MmMaps {
    CUtensorMap a[4], b[3], o[3], dh;
};

template <int CG, int BN, int MODE>
struct MmCfg {
    static constexpr bool kDual = MODE == MM_FWD || MODE == MM_BWD;
    static constexpr bool kBmn = MODE == MM_GRAD;
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
    static_assert(BN == 256 || ((BN == 128 || BN == 384) && kBmn && CG == 2), "384 columns: two MMAs of 256 and 128");
    static constexpr int MMA_N = BN == 384 ? 256 : BN;
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
        gated_pair_grad<ACT, BF>(g[2 * j], g[2 * j + 1], u[2 * j], u[2 * j + 1], widen2<BF>(dh[j]), dg[j], du[j]);
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

template <int CG, int BN, int MODE, bool BF>
__global__ void __launch_bounds__(MmCfg<CG, BN, MODE>::THREADS, 1)
    gated_mm_kernel(const __grid_constant__ MmMaps tm, const __grid_constant__ MmParams p, int* status) {
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
        tzp::tma_prefetch_desc(&tm.a[0]);
        tzp::tma_prefetch_desc(&tm.b[0]);
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
    const int tiles0 = p.g[0].m_tiles * p.g[0].n_tiles * p.g[0].which * p.g[0].splits;
    const int num_tiles = tiles0 + (MODE == MM_GRAD ? p.g[1].m_tiles * p.g[1].n_tiles * p.g[1].which * p.g[1].splits : 0);
    struct Tile {
        int dw, m, n, w, s, kb0, kb1;  // dw: a weights' gradient tile
    };
    const int me = static_cast<int>(blockIdx.x) / CG, team = static_cast<int>(gridDim.x) / CG;
    const int first = p.resident ? static_cast<int>(static_cast<long long>(num_tiles) * me / team) : 0;
    const int last = p.resident ? static_cast<int>(static_cast<long long>(num_tiles) * (me + 1) / team) : 0;
    auto tile_at = [&](int i, Tile& r) -> bool {
        r.dw = 0;
        if (C::kDual && p.resident) {
            const int t = first + i;
            r.n = t / p.g[0].m_tiles;
            r.m = t - r.n * p.g[0].m_tiles;
            r.w = r.s = r.kb0 = 0;
            r.kb1 = p.g[0].kblocks;
            return t < last;
        }
        int t = me + i * team;
        if (t >= num_tiles) return false;
        if (MODE == MM_GRAD && t >= tiles0) {
            r.dw = 1;
            t -= tiles0;
        }
        const Grid& g = p.g[MODE == MM_GRAD ? r.dw : 0];
        const int per = g.m_tiles * g.n_tiles;
        r.s = t / (per * g.which);
        t -= r.s * per * g.which;
        r.w = t / per;
        t -= r.w * per;
        constexpr int GM = 8;
        const int grp = t / (GM * g.n_tiles);
        const int gm = min(GM, g.m_tiles - grp * GM);
        t -= grp * GM * g.n_tiles;
        r.m = grp * GM + t % gm;
        r.n = t / gm;
        r.kb0 = r.s * g.kper;
        r.kb1 = min(g.kblocks, r.kb0 + g.kper);
        return true;
    };
    auto range_at = [&](int i, int& kb0, int& kb1, int& dw) -> bool {  // of tile_at, what the MMA issuer needs
        int t = C::kDual && p.resident ? first + i : me + i * team;
        if (t >= (C::kDual && p.resident ? last : num_tiles)) return false;
        dw = MODE == MM_GRAD && t >= tiles0;
        const Grid& g = p.g[MODE == MM_GRAD ? dw : 0];
        kb0 = 0, kb1 = g.kblocks;
        if (g.splits > 1) {
            kb0 = (dw ? t - tiles0 : t) / (g.m_tiles * g.n_tiles * g.which) * g.kper;
            kb1 = min(g.kblocks, kb0 + g.kper);
        }
        return true;
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
                        if constexpr (MODE == MM_GRAD) {
                            const CUtensorMap* tb;
                            int k = kb * 64;
                            if (q.dw) {
                                const CUtensorMap* ta = &tm.a[2 + q.w];
                                tzp::pair_load_2d<CG>(sa, ta, m0, k, bar);
                                tzp::pair_load_2d<CG>(sa + 8192, ta, m0 + 64, k, bar);
                                tb = &tm.b[2];
                            } else {
                                const bool up = kb >= p.half;
                                if (up) k -= p.half * 64;
                                tzp::pair_load_2d<CG>(sa, &tm.a[up], k, m0, bar);
                                tb = &tm.b[up];
                            }
#pragma unroll
                            for (int j = 0; j < C::BNC / 64; ++j) tzp::pair_load_2d<CG>(sb + j * 8192, tb, b_col(q.n, j), k, bar);
                        } else {
                            tzp::pair_load_2d<CG>(sa, &tm.a[0], kb * 64, m0, bar);
                            if (!need_b) {
                            } else if constexpr (CG == 2) {
                                tzp::pair_load_2d<CG>(sb, &tm.b[rank], kb * 64, q.n * (BN / 2), bar);
                            } else {
                                tzp::pair_load_2d<CG>(sb, &tm.b[0], kb * 64, q.n * (BN / 2), bar);
                                tzp::pair_load_2d<CG>(sb + (BN / 2) * 128, &tm.b[1], kb * 64, q.n * (BN / 2), bar);
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
            constexpr uint32_t idesc0 = tzp::make_idesc(1, BF ? 1 : 0, 128 * CG, C::MMA_N) | (C::kBmn ? 1u << 16 : 0u);
            constexpr uint32_t idesc0_b = tzp::make_idesc(1, BF ? 1 : 0, 128 * CG, 128) | (C::kBmn ? 1u << 16 : 0u);  // columns 256 .. 383
            constexpr uint32_t kBstep = C::kBmn ? 2048u >> 4 : 2u;
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            int kb0, kb1, dw;
            for (int i = 0; ok && range_at(i, kb0, kb1, dw); ++i) {
                const bool amn = MODE == MM_GRAD && dw;  // A is MN-major
                const uint32_t idesc = idesc0 | (amn ? 1u << 15 : 0u), idesc_b = idesc0_b | (amn ? 1u << 15 : 0u);
                const uint32_t a_k = amn ? 2048u >> 4 : 2u;
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
                    const uint64_t ad = amn ? tzp::sdesc_mn128(sa, 8192) : tzp::sdesc_k128(sa);
                    const uint64_t bd = C::kBmn ? tzp::sdesc_mn128(sb, 8192) : tzp::sdesc_k128(sb);
                    if (issue) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t more = (kb > kb0 || k > 0) ? 1u : 0u;
                            tzp::pair_mma_f16<CG>(d, ad + a_k * k, bd + kBstep * k, idesc, more);
                            if constexpr (BN == 384)
                                tzp::pair_mma_f16<CG>(d + 256, ad + a_k * k, bd + (16384u >> 4) + kBstep * k, idesc_b, more);
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
            tzp::tma_load_2d(boxp, &tm.dh, q.n * (BN / 2) + sl * 32, (q.m * CG + static_cast<int>(rank)) * 128 + q4 * 32, &dhbar[e]);
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
                        tzp::tma_store_2d(&tm.o[0], boxp, col0, row0);
                        tzp::bulk_commit();
                    }
                } else {
                    if (store) {
                        tzp::tma_store_2d(&tm.o[1], boxp + 2048, col0, row0);
                        tzp::bulk_commit();
                        tzp::bulk_wait_read<0>();
                    }
                    __syncwarp();
                    stage64<4>(box + 2048, lane, 0, o);
                    tzp::fence_proxy_async();
                    __syncwarp();
                    if (store) {
                        tzp::tma_store_2d(&tm.o[0], boxp + 2048, col0, row0);
                        tzp::bulk_commit();
                    }
                }
            } else {
                constexpr int CH = BN / 64;
                const Grid& g = p.g[q.dw];
                const CUtensorMap* to = &tm.o[g.splits > 1 ? q.dw : q.dw ? 1 + q.w : 0];
                if (lane == 0) tzp::bulk_wait_read<0>();  // the two kinds of tiles use the staging differently
#pragma unroll 1
                for (int c = 0; c < CH; ++c) {
                    const int cc = (sl * CH + c) * 32;
                    const int col0 = q.n * BN + cc;
                    if (col0 >= p.cols) break;
                    uint32_t v[32];
                    tzp::tmem_ld32(td + cc, v);
                    tzp::tmem_ld_wait();
                    if (g.splits > 1) {
                        if (lane == 0) tzp::bulk_wait_read<0>();
                        __syncwarp();
                        stage128(box, lane, v);
                        tzp::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            tzp::tma_store_2d(to, boxp, col0, (q.s * g.which + q.w) * g.m_pad + row0);
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
                            tzp::tma_store_2d(to, boxp + nb * 2048, col0, row0);
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

// Sums partial products [splits][which][m_pad][cols] in order and rounds to 16 bits: up to two jobs of one width.
struct SumJob {
    const float* part;
    void* out[2];
    int which, splits, m_pad, rows;
};
template <bool BF>
__global__ void __launch_bounds__(256) sum_parts_kernel(const __grid_constant__ SumJob j0, const __grid_constant__ SumJob j1, int cols) {
    const long long n0 = static_cast<long long>(j0.rows) * cols / 8, n1 = static_cast<long long>(j1.rows) * cols / 8;
    const long long t0 = n0 * j0.which, total = t0 + n1 * j1.which;
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const SumJob& j = i < t0 ? j0 : j1;
        const long long n8 = i < t0 ? n0 : n1, at = i < t0 ? i : i - t0;
        const int w = at >= n8;
        const long long o = (at - (w ? n8 : 0)) * 8, plane = static_cast<long long>(j.m_pad) * cols;
        float s[8] = {};
        for (int k = 0; k < j.splits; ++k) {
            const float4* src = reinterpret_cast<const float4*>(j.part + (static_cast<long long>(k) * j.which + w) * plane + o);
            const float4 a = __ldcs(src), b = __ldcs(src + 1);
            s[0] += a.x, s[1] += a.y, s[2] += a.z, s[3] += a.w, s[4] += b.x, s[5] += b.y, s[6] += b.z, s[7] += b.w;
        }
        reinterpret_cast<uint4*>(j.out[w])[o / 8] = make_uint4(tzp::pack16x2<BF>(s[0], s[1]), tzp::pack16x2<BF>(s[2], s[3]),
                                                             tzp::pack16x2<BF>(s[4], s[5]), tzp::pack16x2<BF>(s[6], s[7]));
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

template <int CG, int BN, int MODE, bool BF>
int launch_mm(tz_ctx_t ctx, const MmMaps& tm, MmParams p, cudaStream_t s) {
    using C = MmCfg<CG, BN, MODE>;
    auto kern = gated_mm_kernel<CG, BN, MODE, BF>;
    static std::atomic<unsigned> done{0};
    int rc = ensure_smem(kern, C::SMEM, done);
    if (rc) return rc;
    auto count = [](const Grid& g) { return static_cast<long long>(g.m_tiles) * g.n_tiles * g.which * g.splits; };
    const long long tiles = count(p.g[0]) + (MODE == MM_GRAD ? count(p.g[1]) : 0);
    const int groups = (ctx->sm_count - ctx->sm_reserve) / CG;
    const int grid = static_cast<int>(tiles < groups ? tiles : groups) * CG;
    TZ_CHECK(grid > 0, TZ_EINVAL, "gated kernels need %d free SMs", CG);
    p.ring = C::STAGES;
    const int kb = p.g[0].kblocks;
    if (C::kDual && tiles > groups && kb >= 4) {
        // Short sums: the B tiles of a whole column block fit beside a ring of A tiles, and keeping them halves what
        // an SM moves from L2 per tile, which bounds these shapes.  Below 4 K blocks the ring (at most kblocks long)
        // would be too short; above, it has to keep 3 A tiles.
        const int left = (C::BUDGET - kb * C::BNC * 128) / C::A_BYTES;
        int r = left < kb ? left : kb;
        if (r > C::STAGES) r = C::STAGES;
        if (r >= 3) {
            p.resident = 1;
            p.ring = r;
        }
    }
    return launch_cluster(kern, CG, dim3(grid), dim3(C::THREADS), C::SMEM, s, true, tm, p, ctx->d_status);
}

constexpr int kCG = 2, kBN = 256;
// Tokens up to which the forward pass streams weights (gated_rows_kernel).  At 32 tokens it takes 4.7 / 10.0 /
// 14.2 / 26.5 us at (D, F) = (384, 1536) / (1024, 4096) / (2048, 6144) / (4096, 8192), the tiles of 256 tokens 6.3
// / 10.3 / 16.3 / 28.5; with room for 64 tokens it took 6.5 / 14.2 / 16.9 / 29.1.
constexpr int kRowsMax = 32;

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }
size_t a256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// How the gradients' launch is cut: tile width, splits of dx's and the weights' sums, and the workspace's parts.
struct BwdPlan {
    int bn, s_dx, s_dw;
    size_t dgdu, part_dx, part_dw;  // bytes
};

// By an estimate in clocks: every tile's K blocks at the rate its operands arrive at (256 columns: 32 KB per SM and
// K block, 384: 40 KB), the epilogue (beside it, or with one accumulator, 384 columns, after it), the tiles dealt round
// the pairs, and the partial sums' way out and back.  384 columns cover D = 384 in one tile: 18106 tokens, F = 1536
// took 166 us with 256 columns and 148 us with 384.  128 columns give a few tokens more tiles, often enough to do
// without the partial sums and their launch: 77 tokens, D = 384, F = 1000 23.0 us
// with the sums split, 20.7 without.
BwdPlan make_plan(int sms, int64_t T, int64_t D, int64_t F) {
    const int64_t groups = sms / kCG > 0 ? sms / kCG : 1;
    const int64_t mt = ceil_div(T, 128 * kCG), ft = ceil_div(F, 128 * kCG);
    const int kx = 2 * ceil_div(F, 64), kw = ceil_div(T, 64);
    auto splits_ok = [](int kb, int s) { return s == 1 || (kb / s >= 8 && ceil_div(kb, ceil_div(kb, s)) == s); };
    BwdPlan best{};
    double best_cost = 1e300;
    for (int bn = 128; bn <= 384; bn += 128) {
        const int64_t nt = ceil_div(D, bn);
        const double epi = bn == 384 ? 5000.0 : bn == 256 ? 3000.0 : 1700.0;  // an epilogue's own time
        for (int sx = 1; sx <= 16; ++sx) {
            const int64_t nx = mt * nt * sx;
            if (!splits_ok(kx, sx) || (sx > 1 && nx > groups)) continue;
            for (int sw = 1; sw <= 16; ++sw) {
                const int64_t nw = 2 * ft * nt * sw;
                if (!splits_ok(kw, sw) || (sw > 1 && nw > groups)) continue;
                // 24 KB per SM and K block for 128 columns: below the MMA's time only while few SMs ask L2 for it
                const double rate = bn == 384 ? 820.0 : bn == 256 ? 600.0 : nx + nw <= groups / 2 ? 330.0 : 450.0;
                auto tile = [&](int kb) {  // with two accumulators the longer of MMAs and epilogue
                    const double c = kb * rate + 500.0;
                    return bn == 384 ? c + epi : c > epi ? c : epi;
                };
                const double cx = tile(ceil_div(kx, sx)), cw = tile(ceil_div(kw, sw));
                double cost = 0;  // of the slowest pair: pair g has the tiles g, g + groups, ..., dx's first
                const int64_t first[3] = {0, nx % groups, (nx + nw) % groups};  // where the counts step down
                for (int64_t g : first) {
                    const int64_t a = nx > g ? (nx - g - 1) / groups + 1 : 0;
                    const int64_t both = nx + nw > g ? (nx + nw - g - 1) / groups + 1 : 0;
                    const double c = a * cx + (both - a) * cw;
                    if (c > cost) cost = c;
                }
                cost += 3000.0;
                if (sx > 1 || sw > 1)
                    cost += 10000.0 + 8.0 * D * ((sx > 1 ? static_cast<double>(sx) * T : 0.0) + (sw > 1 ? 2.0 * sw * F : 0.0)) / 2500.0;
                if (cost < best_cost) {
                    best_cost = cost;
                    best.bn = bn, best.s_dx = sx, best.s_dw = sw;
                }
            }
        }
    }
    best.dgdu = a256(static_cast<size_t>(T) * F * 2);
    if (best.s_dx > 1) best.part_dx = a256(static_cast<size_t>(best.s_dx) * mt * 128 * kCG * D * 4);
    if (best.s_dw > 1) best.part_dw = a256(static_cast<size_t>(best.s_dw) * 2 * ft * 128 * kCG * D * 4);
    return best;
}
// The last sizes' plan of this thread: a training step asks for the same one again and again.
BwdPlan plan_bwd(int sms, int64_t T, int64_t D, int64_t F) {
    struct Last {
        int sms = 0;
        int64_t T = 0, D = 0, F = 0;
        BwdPlan plan{};
    };
    static thread_local Last last;
    if (last.sms != sms || last.T != T || last.D != D || last.F != F) {
        last.plan = make_plan(sms, T, D, F);
        last.sms = sms, last.T = T, last.D = D, last.F = F;
    }
    return last.plan;
}

// Maps of the dual products: x, Wg and Wu.
template <bool BF>
int dual_maps(MmMaps* tm, const Mat& x, const Mat& wg, const Mat& wu, const Mat& o0, const Mat& o1) {
    const auto S128 = CU_TENSOR_MAP_SWIZZLE_128B, S64 = CU_TENSOR_MAP_SWIZZLE_64B;
    int rc;
    if ((rc = map16<BF>(&tm->a[0], x, 64, 128, S128)) || (rc = map16<BF>(&tm->b[0], wg, 64, kBN / 2, S128)) ||
        (rc = map16<BF>(&tm->b[1], wu, 64, kBN / 2, S128)) || (rc = map16<BF>(&tm->o[0], o0, 32, 32, S64)))
        return rc;
    return o1.p ? map16<BF>(&tm->o[1], o1, 32, 32, S64) : TZ_OK;
}

template <int N, bool BF, bool GRAD>
int launch_rows(tz_ctx_t ctx, const Mat& x, const Mat& wg, const Mat& wu, const Mat& o0, const Mat& o1, const Mat& dh, int act, cudaStream_t s) {
    using C = RowsCfg<N>;
    auto kern = gated_rows_kernel<N, BF, GRAD>;
    static std::atomic<unsigned> done{0};
    int rc = ensure_smem(kern, C::SMEM, done);
    if (rc) return rc;
    CUtensorMap mx, mg, mu;
    const auto S128 = CU_TENSOR_MAP_SWIZZLE_128B;
    if ((rc = map16<BF>(&mx, x, 64, N, S128)) || (rc = map16<BF>(&mg, wg, 64, 128, S128)) || (rc = map16<BF>(&mu, wu, 64, 128, S128))) return rc;
    RowsParams p{};
    const int tiles = ceil_div(o0.cols, 128);
    p.kblocks = ceil_div(x.cols, 64);
    int splits = 1;
    if ((rc = rows_splits<N + GRAD>(kern, C::THREADS, [](int) { return C::SMEM; }, ctx->sm_count - ctx->sm_reserve, tiles, p.kblocks, C::MAX_SPLIT,
                                    &splits)))
        return rc;
    p.kper = ceil_div(p.kblocks, splits);
    p.t = static_cast<int>(x.rows);
    p.f = static_cast<int>(o0.cols);
    p.act = act;
    p.h = const_cast<void*>(o0.p);
    p.du = const_cast<void*>(o1.p);
    p.dh = dh.p;
    p.lddh = dh.ld;
    return rows_launches(ctx, tiles, splits, [&](int t0, int n, bool pdl) {
        p.tile0 = t0;
        return launch_cluster(kern, splits, dim3(splits, n), dim3(C::THREADS), C::SMEM, s, pdl, mx, mg, mu, p, ctx->d_status);
    });
}

// The few-token kernel; *ran says whether the sizes are its own.
template <bool BF, bool GRAD>
int try_rows(tz_ctx_t ctx, const Mat& x, const Mat& wg, const Mat& wu, const Mat& o0, const Mat& o1, const Mat& dh, int act, cudaStream_t s,
             bool* ran) {
    *ran = x.rows <= kRowsMax && o0.cols <= 128 * 65535;  // the grid's second extent
    if (!*ran) return TZ_OK;
    return x.rows <= 16 ? launch_rows<16, BF, GRAD>(ctx, x, wg, wu, o0, o1, dh, act, s)
                        : launch_rows<32, BF, GRAD>(ctx, x, wg, wu, o0, o1, dh, act, s);
}

template <bool BF>
int forward(tz_ctx_t ctx, const Mat& x, const Mat& wg, const Mat& wu, const Mat& h, int act, cudaStream_t s) {
    bool ran = false;
    int rc = try_rows<BF, false>(ctx, x, wg, wu, h, Mat{}, Mat{}, act, s, &ran);
    if (rc || ran) return rc;
    MmMaps tm{};
    if ((rc = dual_maps<BF>(&tm, x, wg, wu, h, Mat{}))) return rc;
    MmParams p{};
    const int kb = ceil_div(x.cols, 64);
    p.g[0] = {ceil_div(x.rows, 128 * kCG), ceil_div(h.cols, kBN / 2), 1, 1, kb, kb, 0};
    p.cols = static_cast<int>(h.cols);
    p.act = act;
    if (x.rows <= 128 && p.g[0].n_tiles > (ctx->sm_count - ctx->sm_reserve) / 2)  // half of a pair's rows would be empty
        return launch_mm<1, kBN, MM_FWD, BF>(ctx, tm, p, s);
    return launch_mm<kCG, kBN, MM_FWD, BF>(ctx, tm, p, s);
}

template <bool BF>
int backward(tz_ctx_t ctx, const Mat& x, const Mat& wg, const Mat& wu, const Mat& dh, const Mat& dx, const Mat& dwg, const Mat& dwu,
             int act, char* ws, cudaStream_t s) {
    const int64_t T = x.rows, D = x.cols, F = dh.cols;
    const BwdPlan b = plan_bwd(ctx->sm_count - ctx->sm_reserve, T, D, F);
    const Mat dg{ws, T, F, F}, du{ws + b.dgdu, T, F, F};
    float* part_dx = reinterpret_cast<float*>(ws + 2 * b.dgdu);
    float* part_dw = reinterpret_cast<float*>(ws + 2 * b.dgdu + b.part_dx);
    const auto S128 = CU_TENSOR_MAP_SWIZZLE_128B, S64 = CU_TENSOR_MAP_SWIZZLE_64B;

    const int mt = ceil_div(T, 128 * kCG), ft = ceil_div(F, 128 * kCG), nt = ceil_div(D, b.bn), kd = ceil_div(D, 64);
    bool ran = false;
    int rc = try_rows<BF, true>(ctx, x, wg, wu, dg, du, dh, act, s, &ran);
    if (rc) return rc;
    if (!ran) {
        MmMaps tm{};
        if ((rc = dual_maps<BF>(&tm, x, wg, wu, dg, du)) || (rc = map16<BF>(&tm.dh, dh, 32, 32, S64))) return rc;
        MmParams p{};
        p.g[0] = {mt, ceil_div(F, kBN / 2), 1, 1, kd, kd, 0};
        p.cols = static_cast<int>(F);
        p.act = act;
        if ((rc = launch_mm<kCG, kBN, MM_BWD, BF>(ctx, tm, p, s))) return rc;
    }

    MmMaps tg{};
    if ((rc = map16<BF>(&tg.a[0], dg, 64, 128, S128)) || (rc = map16<BF>(&tg.a[1], du, 64, 128, S128)) ||
        (rc = map16<BF>(&tg.a[2], dg, 64, 64, S128)) || (rc = map16<BF>(&tg.a[3], du, 64, 64, S128)) ||
        (rc = map16<BF>(&tg.b[0], wg, 64, 64, S128)) || (rc = map16<BF>(&tg.b[1], wu, 64, 64, S128)) ||
        (rc = map16<BF>(&tg.b[2], x, 64, 64, S128)))
        return rc;
    auto part_map = [&](CUtensorMap* m, const float* part, int64_t rows) {
        return encode_tmap_2d_swz(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, part, D, rows, D * 4, 32, 32, S128);
    };
    MmParams q{};
    q.half = ceil_div(F, 64);
    q.g[0] = {mt, nt, 1, b.s_dx, 2 * q.half, ceil_div(2 * q.half, b.s_dx), mt * 128 * kCG};
    const int kt = ceil_div(T, 64);
    q.g[1] = {ft, nt, 2, b.s_dw, kt, ceil_div(kt, b.s_dw), ft * 128 * kCG};
    q.cols = static_cast<int>(D);
    rc = b.s_dx > 1 ? part_map(&tg.o[0], part_dx, static_cast<int64_t>(b.s_dx) * q.g[0].m_pad) : map16<BF>(&tg.o[0], dx, 32, 32, S64);
    if (rc) return rc;
    if (b.s_dw > 1)
        rc = part_map(&tg.o[1], part_dw, 2ll * b.s_dw * q.g[1].m_pad);
    else if (!(rc = map16<BF>(&tg.o[1], dwg, 32, 32, S64)))
        rc = map16<BF>(&tg.o[2], dwu, 32, 32, S64);
    if (rc) return rc;
    rc = b.bn == 384   ? launch_mm<kCG, 384, MM_GRAD, BF>(ctx, tg, q, s)
         : b.bn == 256 ? launch_mm<kCG, 256, MM_GRAD, BF>(ctx, tg, q, s)
                       : launch_mm<kCG, 128, MM_GRAD, BF>(ctx, tg, q, s);
    if (rc || (b.s_dx == 1 && b.s_dw == 1)) return rc;

    SumJob j0{}, j1{};
    if (b.s_dx > 1) j0 = {part_dx, {const_cast<void*>(dx.p), nullptr}, 1, b.s_dx, q.g[0].m_pad, static_cast<int>(T)};
    if (b.s_dw > 1) j1 = {part_dw, {const_cast<void*>(dwg.p), const_cast<void*>(dwu.p)}, 2, b.s_dw, q.g[1].m_pad, static_cast<int>(F)};
    const long long n8 = (static_cast<long long>(j0.rows) * j0.which + static_cast<long long>(j1.rows) * j1.which) * (D / 8);
    const long long blocks = n8 / 256 + 1, most = static_cast<long long>(ctx->sm_count) * 8;
    return launch_kernel(sum_parts_kernel<BF>, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256), 0, s, false, j0, j1,
                         static_cast<int>(D));
}

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
Span span16(const void* p, int64_t rows, int64_t cols, int64_t ld) { return {p, rows, static_cast<size_t>(cols) * 2, static_cast<size_t>(ld) * 2}; }

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
    const size_t wbytes = static_cast<size_t>(d) * f * 2;
    if ((rc = check_apart("tz_gated_linear", "h", h, static_cast<size_t>(t) * f * 2, {span16(x, t, d, ldx), flat(w_gate, wbytes), flat(w_up, wbytes)})))
        return rc;
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
    if (t == 0) {  // an empty sum
        cudaStream_t s = pick_stream(ctx, stream);
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
    const size_t xbytes = static_cast<size_t>(t) * d * 2, wbytes = static_cast<size_t>(d) * f * 2;
    const Span ix = span16(x, t, d, ldx), idh = span16(dh, t, f, lddh), ig = flat(w_gate, wbytes), iu = flat(w_up, wbytes);
    const Span ox = flat(dx, xbytes), og = flat(dw_gate, wbytes), ou = flat(dw_up, wbytes);
    if ((rc = check_apart("tz_gated_linear_backward", "dx", dx, xbytes, {ix, idh, ig, iu})) ||
        (rc = check_apart("tz_gated_linear_backward", "dw_gate", dw_gate, wbytes, {ix, idh, ig, iu, ox})) ||
        (rc = check_apart("tz_gated_linear_backward", "dw_up", dw_up, wbytes, {ix, idh, ig, iu, ox, og})) ||
        (rc = check_apart("tz_gated_linear_backward", "the workspace", workspace, need, {ix, idh, ig, iu, ox, og, ou})))
        return rc;
    cudaStream_t s = pick_stream(ctx, stream);
    const Mat mx{x, t, d, ldx}, mg{w_gate, f, d, d}, mu{w_up, f, d, d}, mdh{dh, t, f, lddh}, mdx{dx, t, d, d}, mwg{dw_gate, f, d, d},
        mwu{dw_up, f, d, d};
    char* ws = static_cast<char*>(workspace);
    return dtype == TZ_PREC_BF16 ? backward<true>(ctx, mx, mg, mu, mdh, mdx, mwg, mwu, act, ws, s)
                                 : backward<false>(ctx, mx, mg, mu, mdh, mdx, mwg, mwu, act, ws, s);
}

}  // extern "C"
