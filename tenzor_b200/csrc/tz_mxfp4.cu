// tz_mxfp4.cu -- microscaled 4-bit floating point (the OCP MXFP4 format): quantiser, and the product of two
// quantised matrices on the block-scaled tensor cores, plain or with the gated epilogue.
//
// Format: blocks of 32 consecutive values of a row share a scale 2^(code - 127) (E8M0, code 255 = NaN); an
// element is E2M1: sign and 0 .5 1 1.5 2 3 4 6.  The scale is 2^(floor(log2 max|x|) - 2), so the largest
// element lands in [4, 8); elements round to nearest, ties to the even code, and saturate at 6.  A block that
// holds a NaN or an infinity gets the NaN scale.
//
// Memory: element codes [rows, cols / 2], two per byte, the even column in the low half.  Scale codes in
// 512-byte chunks of 128 rows x 4 blocks, chunk (r / 128, b / 4) at ((r / 128) * ceil(cols / 128) + b / 4) * 512,
// byte (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4 inside it: the order in which the tensor core's scale
// operand lies in TMEM (lane r % 32, column r / 32, four blocks per 32-bit word), so that one tcgen05.cp moves
// a chunk from shared memory without a rearrangement.
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

constexpr int DT_F32 = TZ_DT_F32, DT_F16 = TZ_DT_F16, DT_BF16 = TZ_DT_BF16;

__host__ __device__ __forceinline__ long long sf_chunk(long long row_block, int k_chunk, int k_chunks) {
    return (row_block * k_chunks + k_chunk) * 512;
}

// ---- quantiser -------------------------------------------------------------------------------------
// Eight consecutive values of a row as loaded: 4 words of 16-bit pairs, or 8 of f32.
template <int DT>
struct Raw8 {
    static constexpr int W = DT == DT_F32 ? 8 : 4;
    uint32_t w[W];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* p, long long i, bool in) {
    Raw8<DT> r;
    uint4 a = make_uint4(0, 0, 0, 0);
    if constexpr (DT == DT_F32) {
        const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
        uint4 b = make_uint4(0, 0, 0, 0);
        if (in) a = __ldg(s), b = __ldg(s + 1);
        r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
    } else {
        if (in) a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i));
    }
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
    return r;
}
template <int DT>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    if constexpr (DT == DT_BF16)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (DT == DT_F32) {
            v[2 * j] = __uint_as_float(r.w[2 * j]), v[2 * j + 1] = __uint_as_float(r.w[2 * j + 1]);
        } else {
            const float2 f = unpack16<DT>(r.w[j]);
            v[2 * j] = f.x, v[2 * j + 1] = f.y;
        }
    }
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// The largest bit pattern of |x|: orders like the value, and an infinity or NaN stays on top.  16-bit values are
// compared as packed 15-bit patterns (top8), and only the largest is widened to f32 (top_f32).
template <int DT>
__device__ __forceinline__ uint32_t top8(const Raw8<DT>& r) {
    uint32_t t = 0;
#pragma unroll
    for (int j = 0; j < Raw8<DT>::W; ++j) t = DT == DT_F32 ? max(t, r.w[j] & 0x7FFFFFFFu) : max_u16x2(t, r.w[j] & 0x7FFF7FFFu);
    return t;
}
template <int DT>
__device__ __forceinline__ uint32_t top_max(uint32_t a, uint32_t b) {
    return DT == DT_F32 ? max(a, b) : max_u16x2(a, b);
}
template <int DT>
__device__ __forceinline__ uint32_t top_f32(uint32_t t) {
    if constexpr (DT == DT_F32) return t;
    const uint32_t m = max(t & 0xFFFFu, t >> 16);
    if constexpr (DT == DT_BF16) return m << 16;
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
}
// The scale code for the largest |x| (f32 bits), and 1 / scale.
__device__ __forceinline__ uint32_t scale_of(uint32_t top, float& inv) {
    const uint32_t e = top >> 23;  // floor(log2) + 127; 0 for subnormals, whose scale is the smallest anyway
    const uint32_t sc = e > 2u ? e - 2u : 0u;
    inv = __uint_as_float((254u - sc) << 23);
    return e == 255u ? 255u : sc;
}

// Eight values to eight E2M1 codes (value j in bits 4j .. 4j+3).
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8], float inv) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv), "f"(v[6] * inv),
          "f"(v[7] * inv));
    return r;
}

template <int DT>
__device__ __forceinline__ uint32_t encode8(const Raw8<DT>& r, float inv) {
    float v[8];
    widen8<DT>(r, v);
    return e2m1x8(v, inv);
}
// Quantises a block spread over 4 neighbouring lanes (8 values each); returns the codes, `sc` the scale code.
template <int DT>
__device__ __forceinline__ uint32_t quant_block(const Raw8<DT>& r, uint32_t& sc) {
    uint32_t top = top8<DT>(r);
    top = top_max<DT>(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = top_max<DT>(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    float inv;
    sc = scale_of(top_f32<DT>(top), inv);
    return encode8<DT>(r, inv);
}

// A warp quantises 1024 columns of a row, a lane 16 values at a time (two lanes make a block), its four loads in flight
// together.  Bound by HBM at 2 (or 4) bytes read and 0.53 written per value: 8192 x 8192 bf16 takes 28 us, 6.0 TB/s.
// With 8 values a lane and four lanes a block the ALU was the bound (13 instructions a value, 37 us).
// Row r of x becomes row r of the result, or with GROUP > 0 row (r / GROUP) * 2 GROUP + r % GROUP + off, which
// interleaves two matrices in groups of GROUP rows.
template <int DT, int GROUP>
__global__ void __launch_bounds__(256) quantize_mxfp4_kernel(const void* x, long long ldx, uint8_t* codes, uint8_t* scales, long long rows,
                                                             int cols, int off) {
    const int lane = threadIdx.x & 31;
    const int k_chunks = (cols + 127) / 128;
    const int c0 = static_cast<int>(blockIdx.x) * 1024 + lane * 16;
    for (long long r = blockIdx.y * 8ll + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8ll) {
        Raw8<DT> v[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) v[j][h] = load8<DT>(x, r * ldx + c0 + 512 * j + 8 * h, c0 + 512 * j < cols);
        const long long ro = GROUP > 0 ? (r / GROUP) * (2 * GROUP) + r % GROUP + off : r;
        uint8_t* crow = codes + ((ro * cols + c0) >> 1);
        uint8_t* srow = scales + sf_chunk(ro >> 7, c0 >> 7, k_chunks) + (ro & 31) * 16 + ((ro & 127) >> 5) * 4 + ((c0 >> 5) & 3);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t top = top_max<DT>(top8<DT>(v[j][0]), top8<DT>(v[j][1]));
            top = top_max<DT>(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            float inv;
            const uint32_t sc = scale_of(top_f32<DT>(top), inv);
            const int c = c0 + 512 * j;
            if (c < cols) {
                *reinterpret_cast<uint2*>(crow + 256 * j) = make_uint2(encode8<DT>(v[j][0], inv), encode8<DT>(v[j][1], inv));
                if ((lane & 1) == 0) srow[2048 * j] = static_cast<uint8_t>(sc);
            }
            // The last word of a row that ends inside it: 0 for the blocks past the end.
            if (c >= cols && (lane & 1) == 0 && (c >> 7) < k_chunks) srow[2048 * j] = 0;
        }
    }
    tzp::pdl_trigger();  // the product that follows may set up
}

// 2^(code - 127) in f32 (code 0 is the subnormal 2^-127, 255 a NaN).
__device__ __forceinline__ float e8m0(uint32_t code) {
    return __uint_as_float(code == 255u ? 0x7FC00000u : code == 0u ? 0x00400000u : code << 23);
}

// Two E2M1 codes (low nibble first) as f32.
__device__ __forceinline__ float2 e2m1x2(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 t, u;\n\t.reg .b16 s;\n\tcvt.u16.u32 s, %1;\n\tmov.b16 {t, u}, s;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The quantiser's split the other way round.
template <int DT>
__global__ void __launch_bounds__(256) dequantize_mxfp4_kernel(const uint8_t* codes, const uint8_t* scales, void* out, long long rows, int cols) {
    const int lane = threadIdx.x & 31;
    const int k_chunks = (cols + 127) / 128;
    const int c0 = static_cast<int>(blockIdx.x) * 1024 + lane * 8;
    for (long long r = blockIdx.y * 8ll + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8ll) {
        const uint8_t* srow = scales + sf_chunk(r >> 7, 0, k_chunks) + (r & 31) * 16 + ((r & 127) >> 5) * 4;
        uint32_t q[4], sc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + 256 * j;
            if (c < cols) {
                q[j] = __ldg(reinterpret_cast<const uint32_t*>(codes + (r * cols + c) / 2));
                sc[j] = __ldg(srow + (c >> 7) * 512 + ((c >> 5) & 3));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + 256 * j;
            if (c >= cols) break;
            const float s = e8m0(sc[j]);
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = e2m1x2((q[j] >> (8 * e)) & 255u);
                v[2 * e] = f.x * s, v[2 * e + 1] = f.y * s;
            }
            if constexpr (DT == DT_F32) {
                float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + r * cols + c);
                o[0] = make_float4(v[0], v[1], v[2], v[3]);
                o[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                constexpr bool BF = DT == DT_BF16;
                *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + r * cols + c) =
                    make_uint4(tzp::pack16x2<BF>(v[0], v[1]), tzp::pack16x2<BF>(v[2], v[3]), tzp::pack16x2<BF>(v[4], v[5]),
                               tzp::pack16x2<BF>(v[6], v[7]));
            }
        }
    }
}

// ---- block-scaled product --------------------------------------------------------------------------
// y = q(x) q(W)^T (+ bias), or with GATED the gated form of interleaved weights: W rows come as 16 gate rows,
// 16 up rows, and so on, so a 32-column chunk of the accumulator holds the gate and the up values of 16 outputs.
//
// The structure of the 16-bit gated kernel (persistent, TMA producer, MMA issuer, epilogue warps in groups of 12, two
// accumulators, CTA pairs).  A K block is 128 bytes = 256 values: four MMAs of 64.  Its scales are two chunks for the
// CTA's 128 rows of A and four for the columns' rows of W (both CTAs of a pair keep all of them).  They go to TMEM by
// tcgen05.cp, each stage to its own 24 columns: a stage's scales are only replaced once its MMAs have completed.
// BN = 192 leaves TMEM for that: 2 x 192 + 24 x stages <= 512 columns.
//
// Measured: 8192 x 8192 x 8192 f16 196 us alone (5.6 PFLOP/s, tensor pipe 77 % active; the feed from L2, 31 KB per SM
// for 384 clocks of MMAs, is the bound), about 240 us in a loop under the power cap.  The issue of a K block's six
// scale copies and four MMAs is serial: with a branch on the lane number around it (operands moved to uniform
// registers one by one) a K block took 1050 clocks and the product 355 us.  The encoder batch's gated form (T 18106,
// D 384, F 1536) takes 26 us: two K blocks a tile, bound by the epilogue (special-function unit 61 %; 31 us with one
// group of epilogue warps for both accumulators).
constexpr int GROUP = 16;

struct MxParams {
    int m_tiles, n_tiles;
    int n;              // columns of the output before the gate
    int k_chunks;       // scale chunks per row block
    int k;              // values
    const float* bias;
    int act;
};

template <int CG, bool GATED>
struct MxCfg {
    static constexpr int BN = 192;
    // A group of 12 epilogue warps reads an accumulator: 4 TMEM lane quarters x 3 slices of 64 columns.  The gated
    // form, bound by its exponentials, has a group for each of the two accumulators, so that one group's loads and
    // stores run under the other's arithmetic.
    static constexpr int GROUPS = GATED ? 2 : 1;
    static constexpr int EPI = 12 * GROUPS;
    static constexpr int THREADS = 64 + 32 * EPI;
    static constexpr int BNC = BN / CG;
    static constexpr int A_BYTES = 128 * 128;
    static constexpr int B_BYTES = BNC * 128;
    static constexpr int SF_BYTES = 3072;  // A: 2 chunks; B: 2 row blocks x 2 chunks
    static constexpr int STAGE = A_BYTES + B_BYTES + SF_BYTES;
    static constexpr int BOX = GATED ? 2048 : 4096;  // staging of one epilogue warp
    static constexpr int STAGING = EPI * BOX;
    static constexpr int STAGES = CG == 2 ? 5 : 4;
    static constexpr int SF_COLS = 24;
    static constexpr int SF0 = 2 * BN;
    static constexpr int SMEM = STAGES * STAGE + STAGING + 512 + 1024;
    static_assert(SF0 + STAGES * SF_COLS <= 512, "TMEM");
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(STAGE % 1024 == 0, "swizzle atoms");
};

// kind::mxf4 instruction descriptor: E2M1 operands (1), E8M0 scales (bit 23), K-major, scale ids of A and B.
__host__ __device__ constexpr uint32_t mx_idesc(uint32_t M, uint32_t N, uint32_t sf_id) {
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 4) << 24) | (sf_id << 29);
}

template <int CG>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// One 512-byte scale chunk (32 rows of 16 bytes) to 4 TMEM columns, repeated in the four lane quarters.
template <int CG>
__device__ __forceinline__ void sf_copy(uint32_t taddr, uint32_t smem_addr) {
    uint64_t d = 0;  // no swizzle: 8-row groups 128 bytes apart
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(128 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    if constexpr (CG == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

template <int CG, int OUT, bool GATED>
__global__ void __launch_bounds__(MxCfg<CG, GATED>::THREADS, 1)
    mxfp4_mm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmO,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const MxParams p, int* status) {
    using C = MxCfg<CG, GATED>;
    constexpr int STAGES = C::STAGES, BN = C::BN;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = tzp::smem_u32(smem_raw);
    uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
    uint8_t* staging = smem + STAGES * C::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
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
            tzp::mbar_init(&tempty[a], 12 * CG);
        }
        tzp::mbar_init(drain, 1);
        *abort_flag = 0;
        tzp::fence_mbar_init();
        tzp::tma_prefetch_desc(&tmA);
        tzp::tma_prefetch_desc(&tmB);
    }
    if (warp == 1) tzp::pair_tmem_alloc<CG>(tmem_slot, 512);
    tzp::tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) tzp::cluster_sync();
    tzp::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    tzp::pdl_wait();

    const int num_tiles = p.m_tiles * p.n_tiles;
    const int kblocks = (p.k + 255) / 256;
    auto tile_of = [&](int t, int& m, int& n) {  // groups of 8 row blocks walk the column blocks together
        constexpr int GM = 8;
        const int grp = t / (GM * p.n_tiles);
        const int gm = min(GM, p.m_tiles - grp * GM);
        t -= grp * GM * p.n_tiles;
        m = grp * GM + t % gm;
        n = t / gm;
    };
    const int t0 = static_cast<int>(blockIdx.x) / CG, tstep = static_cast<int>(gridDim.x) / CG;

    if (warp == 0) {
        {
            // ---- TMA producer (the whole warp; one lane issues) ----
            const bool issue = tzp::elect_one();
            int stage = 0;
            uint32_t phase = 0, armed = 0, armed_par = 0;
            bool ok = true;
            for (int t = t0; ok && t < num_tiles; t += tstep) {
                int m, n;
                tile_of(t, m, n);
                const int mb = m * CG + static_cast<int>(rank);
                const int nb = n * BN / 128;
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!tzp::warp_wait(&empty[stage], phase ^ 1u, status, abort_flag)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) {
                        armed |= 1u << stage;
                        armed_par = (armed_par & ~(1u << stage)) | (phase << stage);
                    }
                    const uint32_t bar = CG == 2 ? tzp::mapa(&full[stage], 0) : tzp::smem_u32(&full[stage]);
                    const uint32_t sa = tzp::smem_u32(smem + stage * C::STAGE);
                    const uint32_t sb = sa + C::A_BYTES, sf = sb + C::B_BYTES;
                    if (issue) {
                        if (rank == 0) tzp::mbar_arrive_expect_tx(&full[stage], CG * C::STAGE);
                        tzp::pair_load_2d<CG>(sa, &tmA, kb * 128, mb * 128, bar);
                        tzp::pair_load_2d<CG>(sb, &tmB, kb * 128, n * BN + static_cast<int>(rank) * C::BNC, bar);
                        // two chunks each (past a row block's last chunk: of the next one or zeros, which no MMA uses)
                        tzp::pair_load_2d<CG>(sf, &tmSA, 0, mb * p.k_chunks + 2 * kb, bar);
                        tzp::pair_load_2d<CG>(sf + 1024, &tmSB, 0, nb * p.k_chunks + 2 * kb, bar);
                        tzp::pair_load_2d<CG>(sf + 2048, &tmSB, 0, (nb + 1) * p.k_chunks + 2 * kb, bar);
                    }
                    __syncwarp();
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            for (int s = 0; s < STAGES; ++s)  // every copy has landed before the CTA can exit (bounded)
                if (armed & (1u << s)) tzp::mbar_wait(&full[s], (armed_par >> s) & 1u, status, nullptr);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            // ---- MMA issuer (the whole warp; one lane issues) ----
            const bool issue = tzp::elect_one();
            constexpr uint32_t idesc0 = mx_idesc(128 * CG, BN, 0), idesc2 = mx_idesc(128 * CG, BN, 2);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int t = t0; ok && t < num_tiles; t += tstep) {
                int m, n;
                tile_of(t, m, n);
                if (!tzp::warp_wait(&tempty[acc], acc_phase ^ 1u, status, abort_flag)) break;
                tzp::tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                const uint32_t boff = static_cast<uint32_t>((n * BN & 127) / 32);  // the tile's first row inside its scale chunk
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!tzp::warp_wait(&full[stage], phase, status, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tzp::tc_fence_after();
                    const uint32_t sa = tzp::smem_u32(smem + stage * C::STAGE);
                    const uint32_t sf = sa + C::A_BYTES + C::B_BYTES;
                    const uint32_t tsf = tmem_base + static_cast<uint32_t>(C::SF0 + stage * C::SF_COLS);
                    const int left = p.k - kb * 256;
                    const uint64_t ad = tzp::sdesc_k128(sa), bd = tzp::sdesc_k128(sa + C::A_BYTES);
                    // TMEM columns of the stage: A chunk 0 (4), A chunk 1 (4), B chunk 0 (8), B chunk 1 (8)
                    if (left >= 256) {
                        if (issue) {
                            sf_copy<CG>(tsf, sf);
                            sf_copy<CG>(tsf + 8, sf + 1024);
                            sf_copy<CG>(tsf + 12, sf + 2048);
                            sf_copy<CG>(tsf + 4, sf + 512);
                            sf_copy<CG>(tsf + 16, sf + 1536);
                            sf_copy<CG>(tsf + 20, sf + 2560);
                            mx_mma<CG>(d, ad, bd, idesc0, tsf, tsf + 8 + boff, kb != 0 ? 1u : 0u);
                            mx_mma<CG>(d, ad + 2u, bd + 2u, idesc2, tsf, tsf + 8 + boff, 1u);
                            mx_mma<CG>(d, ad + 4u, bd + 4u, idesc0, tsf + 4, tsf + 16 + boff, 1u);
                            mx_mma<CG>(d, ad + 6u, bd + 6u, idesc2, tsf + 4, tsf + 16 + boff, 1u);
                            tzp::pair_commit<CG>(&empty[stage]);
                        }
                    } else if (issue) {  // the last values of a row
                        sf_copy<CG>(tsf, sf);
                        sf_copy<CG>(tsf + 8, sf + 1024);
                        sf_copy<CG>(tsf + 12, sf + 2048);
                        if (left > 128) {
                            sf_copy<CG>(tsf + 4, sf + 512);
                            sf_copy<CG>(tsf + 16, sf + 1536);
                            sf_copy<CG>(tsf + 20, sf + 2560);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k == 0 || left > 64 * k)
                                mx_mma<CG>(d, ad + 2u * k, bd + 2u * k, (k & 1) ? idesc2 : idesc0, tsf + 4 * (k >> 1),
                                           tsf + 8 + 8 * (k >> 1) + boff, (kb | k) != 0 ? 1u : 0u);
                        tzp::pair_commit<CG>(&empty[stage]);
                    }
                    __syncwarp();
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (issue) tzp::pair_commit<CG>(&tfull[acc]);
                __syncwarp();
                if (++acc == 2) {
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
        // ---- epilogue: TMEM lane quarter (warp % 4), 64 of the columns ----
        const int e = warp - 2, q4 = warp & 3, grp = e / 12, sl = (e - grp * 12) >> 2;
        const uint32_t box = tzp::smem_u32(staging) + static_cast<uint32_t>(e * C::BOX);
        uint8_t* boxp = staging + e * C::BOX;
        int acc = grp;  // two groups: each keeps to its accumulator and takes every other tile
        uint32_t acc_phase = 0;
        for (int t = t0 + grp * tstep; t < num_tiles; t += C::GROUPS * tstep) {
            int m, n;
            tile_of(t, m, n);
            if (t + C::GROUPS * tstep >= num_tiles) tzp::pdl_trigger();
            if (!tzp::warp_wait(&tfull[acc], acc_phase, status, abort_flag)) break;
            tzp::tc_fence_after();
            const uint32_t td = tmem_base + (static_cast<uint32_t>(q4 * 32) << 16) + static_cast<uint32_t>(acc * BN + sl * 64);
            const int row0 = (m * CG + static_cast<int>(rank)) * 128 + q4 * 32;
            const int colt = n * BN + sl * 64;
            if (lane == 0) tzp::bulk_wait_read<0>();  // the previous tile's stores have read the boxes
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col0 = colt + 32 * c;
                uint32_t v[32];
                tzp::tmem_ld32(td + 32 * c, v);
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
                if constexpr (GATED) {
                    uint32_t o[8];
#define TZ_G(A) \
    for (int j = 0; j < 8; ++j) o[j] = gated_pair<A, OUT == DT_BF16>(v[2 * j], v[2 * j + 1], v[16 + 2 * j], v[17 + 2 * j])
                    TZ_ACT_SWITCH(p.act, _Pragma("unroll") TZ_G)
#undef TZ_G
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        tzp::st_shared_v4(box + lane * 64 + (((2 * c + u) ^ ((lane >> 1) & 3)) << 4), o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                    continue;
                }
                if (p.bias) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if (col0 + j < p.n) {  // n is a multiple of 8
                            const float4 b4 = __ldg(reinterpret_cast<const float4*>(p.bias + col0 + j));
                            v[j] = __float_as_uint(__uint_as_float(v[j]) + b4.x);
                            v[j + 1] = __float_as_uint(__uint_as_float(v[j + 1]) + b4.y);
                            v[j + 2] = __float_as_uint(__uint_as_float(v[j + 2]) + b4.z);
                            v[j + 3] = __float_as_uint(__uint_as_float(v[j + 3]) + b4.w);
                        }
                    }
                }
                if constexpr (OUT == DT_F32) {  // one box of 32 columns, stored at once
                    if (c == 1) {
                        if (lane == 0) tzp::bulk_wait_read<0>();
                        __syncwarp();
                    }
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        tzp::st_shared_v4(box + lane * 128 + ((u ^ (lane & 7)) << 4), v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
                    tzp::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0 && col0 < p.n) {
                        tzp::tma_store_2d(&tmO, boxp, col0, row0);
                        tzp::bulk_commit();
                    }
                } else if constexpr (!GATED) {
                    uint32_t o[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = tzp::pack16x2<OUT == DT_BF16>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        tzp::st_shared_v4(box + c * 2048 + lane * 64 + ((u ^ ((lane >> 1) & 3)) << 4), o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                }
            }
            if constexpr (OUT != DT_F32) {
                tzp::fence_proxy_async();
                __syncwarp();
                if (lane == 0 && colt < p.n) {
                    if constexpr (GATED) {
                        tzp::tma_store_2d(&tmO, boxp, colt / 2, row0);
                    } else {
                        tzp::tma_store_2d(&tmO, boxp, colt, row0);
                        if (colt + 32 < p.n) tzp::tma_store_2d(&tmO, boxp + 2048, colt + 32, row0);
                    }
                    tzp::bulk_commit();
                }
            }
            if (C::GROUPS == 2) {
                acc_phase ^= 1u;
            } else if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        tzp::pdl_trigger();  // a group without a tile
        if (lane == 0) tzp::bulk_wait_all();
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
        tzp::pair_tmem_dealloc<CG>(tmem_base, 512);
    }
}

// ---- few rows (serving) ----------------------------------------------------------------------------
// The product for up to 32 rows of x, bound by reading the 4-bit weights once.  As in gated_rows_kernel the weights
// are the A operand (128 of their rows: M) and the rows of x the B operand (N = 16 or 32), and the K blocks of a
// tile are split over a cluster.  x is quantised inside the kernel, straight into the MMA's operand layout: each
// CTA needs its K slice only, so the work (0.5 us for 16 rows of 4096) hides behind the first weight copies and the
// separate quantiser launch goes away.  With GATED a warp's 32 TMEM lanes are 16 gate rows and their 16 up rows.
//
// Measured (a call of a graph, bf16; weights from HBM: 12 sets of them in turn, 213 MB or more / from L2: one set): D 4096,
// 2 F 16384 gated 11.0 / 6.9 us for one row, 12.4 / 8.8 for 16, 15.2 / 12.2 for 32; K 4096, N 8192 8.0 us from HBM for one
// row, 8.5 / 6.6 for 16, 10.2 / 8.8 for 32.  What is left over the weights' own time from HBM (5.4 and 2.7 us) is the
// launch and the first copies (about 4 us) and, from 16 rows on, the quantising.
struct MxRowsParams {
    const void* x;
    long long ldx;
    void* y;
    const float* bias;
    int rows, k, n;      // of x, of a row, weight rows
    int k_chunks, kblocks, kper;
    int tile0;           // the launch's first tile of weight rows
    int act;
};

template <int N>
struct MxRowsCfg {
    static constexpr int QWARPS = N == 32 ? 16 : 8;  // two rows of a K block each
    static constexpr int THREADS = 96 + 32 * QWARPS;
    static constexpr int STAGE = 16384 + 1024;
    static constexpr int STAGES = 4;             // even: a stage's K blocks belong to one MMA issuer
    static constexpr int SF_COLS = 16;           // per stage: A 2 x 4, B 2 x 4
    static constexpr int SF0 = 64;
    static constexpr int TCOLS = 128;            // two accumulators of 32, 4 * 16 columns of scales
    static constexpr int B_KB = N * 128 + 1024;  // one K block of x: codes and two scale chunks
    static constexpr int PART = 128 * N * 4;
    static constexpr int MAX_SPLIT = 1 + STAGES * STAGE / PART;
    static constexpr int MAX_KB = (227 * 1024 - 2048 - STAGES * STAGE) / B_KB < 32 ? (227 * 1024 - 2048 - STAGES * STAGE) / B_KB : 32;
    static constexpr int smem(int kper) { return STAGES * STAGE + kper * B_KB + 1024 + 1024; }
};

template <int N, int XDT, int OUT, bool GATED>
__global__ void __launch_bounds__(MxRowsCfg<N>::THREADS, 1)
    mxfp4_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmSW, const MxRowsParams p, int* status) {
    using C = MxRowsCfg<N>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (tzp::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* xq = smem + STAGES * C::STAGE;  // [K block][codes N x 128 swizzled | 2 scale chunks]
    uint64_t* full = reinterpret_cast<uint64_t*>(xq + p.kper * C::B_KB);
    uint64_t* empty = full + STAGES;
    uint64_t* done = empty + STAGES;
    uint64_t* xready = done + 1;  // one per K block of this CTA (at most 32)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(xready + 32);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(tzp::cluster_ctarank());
    const int tile = p.tile0 + static_cast<int>(blockIdx.y), n0 = tile * 128;
    const int kb0 = rank * p.kper, kb1 = min(p.kblocks, kb0 + p.kper);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tzp::mbar_init(&full[s], 1);
            tzp::mbar_init(&empty[s], 1);
        }
        tzp::mbar_init(done, 2);
        for (int i = 0; i < 32; ++i) tzp::mbar_init(&xready[i], C::QWARPS);
        *abort_flag = 0;
        tzp::fence_mbar_init();
        tzp::tma_prefetch_desc(&tmW);
        tzp::tma_prefetch_desc(&tmSW);
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
                    tzp::tma_load_2d(a, &tmW, kb * 128, n0, &full[s]);
                    tzp::tma_load_2d(a + 16384, &tmSW, 0, tile * p.k_chunks + 2 * kb, &full[s]);
                }
                __syncwarp();
            }
            for (int s = 0; s < STAGES; ++s)  // every copy has landed before the stages are used again (bounded)
                if (armed & (1u << s)) tzp::mbar_wait(&full[s], (armed_par >> s) & 1u, status, nullptr);
        }
    } else if (warp == 1 || warp == 2 + C::QWARPS) {
        // Two MMA issuers (whole warps; one lane issues) take the K blocks in turn, each with an accumulator of its own:
        // the issue of a K block's scale copies and MMAs is serial, and the tensor core idles for most of it.
        {
            const bool issue = tzp::elect_one();
            const int mi = warp == 1 ? 0 : 1;
            const uint32_t d = tmem_base + 32u * mi;
            constexpr uint32_t idesc0 = mx_idesc(128, N, 0), idesc2 = mx_idesc(128, N, 2);
            for (int kb = kb0 + mi, i = mi; kb < kb1; kb += 2, i += 2) {
                const int s = i % STAGES;
                if (!tzp::warp_wait(&xready[i], 0, status, abort_flag)) break;
                if (!tzp::warp_wait(&full[s], (i / STAGES) & 1, status, abort_flag)) break;
                tzp::tc_fence_after();
                const uint32_t a = tzp::smem_u32(smem + s * C::STAGE), b = tzp::smem_u32(xq + i * C::B_KB);
                const uint32_t tsf = tmem_base + static_cast<uint32_t>(C::SF0 + s * C::SF_COLS);
                const int left = p.k - kb * 256;
                const uint64_t ad = tzp::sdesc_k128(a), bd = tzp::sdesc_k128(b);
                if (issue) {
                    sf_copy<1>(tsf, a + 16384);
                    sf_copy<1>(tsf + 8, b + N * 128);
                    if (left > 128) {
                        sf_copy<1>(tsf + 4, a + 16384 + 512);
                        sf_copy<1>(tsf + 12, b + N * 128 + 512);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k == 0 || left > 64 * k)
                            mx_mma<1>(d, ad + 2u * k, bd + 2u * k, (k & 1) ? idesc2 : idesc0, tsf + 4 * (k >> 1), tsf + 8 + 4 * (k >> 1),
                                      (i > mi || k != 0) ? 1u : 0u);
                    tzp::umma_commit(&empty[s]);
                }
                __syncwarp();
            }
            if (issue) tzp::umma_commit(done);
            __syncwarp();
            tzp::mbar_wait(done, 0, status, nullptr);
        }
    } else {
        // ---- quantise this CTA's K slice of x, one K block (256 values of N rows) after the other; a warp takes
        // two rows of the block, a lane 8 values of each.  Rows past the last one are zeros with the smallest scale.
        // The next block's values are on their way while a block is quantised. ----
        constexpr int R = N / C::QWARPS;
        Raw8<XDT> v[R];
        auto fetch = [&](int kb) {
            const int c = kb * 256 + lane * 8;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int r = warp - 2 + j * C::QWARPS;
                v[j] = load8<XDT>(p.x, r * p.ldx + c, r < p.rows && c < p.k);
            }
        };
        fetch(kb0);
        for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
            uint8_t* blk = xq + i * C::B_KB;
            Raw8<XDT> u[R];
#pragma unroll
            for (int j = 0; j < R; ++j) u[j] = v[j];
            if (kb + 1 < kb1) fetch(kb + 1);
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const int r = warp - 2 + j * C::QWARPS;
                uint32_t q = 0, w = 0;
                if (r < p.rows) {  // the same for the whole warp
                    uint32_t sc;
                    q = quant_block<XDT>(u[j], sc);
                    w = sc << (8 * ((lane >> 2) & 3));
                    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 4);
                    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 8);
                }
                // 4 bytes at byte 4 * lane of a 128-byte row, 128-byte swizzle (16-byte unit u at u ^ (r % 8))
                *reinterpret_cast<uint32_t*>(blk + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = q;
                if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(blk + N * 128 + (lane >> 4) * 512 + r * 16) = w;
            }
            tzp::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tzp::mbar_arrive(&xready[i]);
        }
    }
    // All products of this CTA are in its TMEM and its stages are free; then the same of every CTA.
    tzp::tc_fence_before();
    __syncthreads();
    const bool split = p.kper < p.kblocks;
    if (split) tzp::cluster_sync();
    tzp::tc_fence_after();

    const int q4 = warp & 3, row = q4 * 32 + lane;  // weight row n0 + row
    float* part = reinterpret_cast<float*>(smem);   // [rank - 1][N][128]
    const uint32_t td = tmem_base + (static_cast<uint32_t>(q4 * 32) << 16);
    const bool epi = warp >= 2 && warp < 6, two = kb1 - kb0 > 1;
    auto sums = [&](int c, uint32_t (&v)[16]) {  // 16 columns of both accumulators
        uint32_t w[16];
        tzp::tmem_ld16(td + c, v);
        tzp::tmem_ld16(td + 32 + c, w);
        tzp::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (two) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(w[j]));
    };
    if (rank > 0 && epi) {
        const uint32_t dst = tzp::mapa(part + (rank - 1) * N * 128 + row, 0);
#pragma unroll 1
        for (int c = 0; c < N; c += 16) {
            uint32_t v[16];
            sums(c, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) st_cluster_f32(dst + (c + j) * 512, __uint_as_float(v[j]));
        }
    }
    if (split) tzp::cluster_sync();
    if (rank == 0 && epi) {
        const int ranks = (p.kblocks + p.kper - 1) / p.kper;
        const float bias = !GATED && p.bias && n0 + row < p.n ? __ldg(p.bias + n0 + row) : 0.0f;
#pragma unroll 1
        for (int c = 0; c < N; c += 16) {
            if (c >= p.rows) break;
            uint32_t v[16];
            sums(c, v);
            for (int r = 1; r < ranks; ++r) {
                const float* src = part + (r - 1) * N * 128 + row;
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + src[(c + j) * 128]);
            }
            if constexpr (GATED) {
                uint32_t u[16], o[8];
#pragma unroll
                for (int j = 0; j < 16; ++j) u[j] = __shfl_down_sync(0xFFFFFFFFu, v[j], 16);
#define TZ_G(A) \
    for (int j = 0; j < 8; ++j) o[j] = gated_pair<A, OUT == DT_BF16>(v[2 * j], v[2 * j + 1], u[2 * j], u[2 * j + 1])
                TZ_ACT_SWITCH(p.act, _Pragma("unroll") TZ_G)
#undef TZ_G
                const int f = (n0 + q4 * 32) / 2 + lane;
                if (lane < 16 && 2 * f < p.n) {
                    uint16_t* out = reinterpret_cast<uint16_t*>(p.y) + f;
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (c + j < p.rows) out[static_cast<long long>(c + j) * (p.n / 2)] = static_cast<uint16_t>(o[j / 2] >> (16 * (j & 1)));
                }
            } else if (n0 + row < p.n) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (c + j >= p.rows) break;
                    const float y = p.bias ? __uint_as_float(v[j]) + bias : __uint_as_float(v[j]);
                    const long long o = static_cast<long long>(c + j) * p.n + n0 + row;
                    if constexpr (OUT == DT_F32)
                        reinterpret_cast<float*>(p.y)[o] = y;
                    else if constexpr (OUT == DT_F16)
                        reinterpret_cast<__half*>(p.y)[o] = __float2half_rn(y);
                    else
                        reinterpret_cast<__nv_bfloat16*>(p.y)[o] = __float2bfloat16_rn(y);
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

constexpr int kCG = 2;
constexpr int kRowsMax = 32;  // rows up to which the product streams weights (mxfp4_rows_kernel)

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

struct Q4 {
    const uint8_t* codes;
    const uint8_t* scales;
    int64_t rows;
};

template <int CG, int OUT, bool GATED>
int launch_mx_cg(tz_ctx_t ctx, const Q4& a, const Q4& b, int k, const float* bias, void* y, int act, cudaStream_t s) {
    using C = MxCfg<CG, GATED>;
    auto kern = mxfp4_mm_kernel<CG, OUT, GATED>;
    static std::atomic<unsigned> done{0};
    int rc = ensure_smem(kern, C::SMEM, done);
    if (rc) return rc;
    CUtensorMap ma, mb, mo, msa, msb;
    const auto S128 = CU_TENSOR_MAP_SWIZZLE_128B, S0 = CU_TENSOR_MAP_SWIZZLE_NONE;
    const int kc = ceil_div(k, 128);  // scale chunks: rows of 128 words
    if ((rc = encode_tmap_2d_swz(&msa, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, a.scales, 128, static_cast<uint64_t>(ceil_div(a.rows, 128)) * kc, 512, 128, 2, S0)) ||
        (rc = encode_tmap_2d_swz(&msb, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, b.scales, 128, static_cast<uint64_t>(ceil_div(b.rows, 128)) * kc, 512, 128, 2, S0)))
        return rc;
    if ((rc = encode_tmap_2d_swz(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.codes, k / 2, a.rows, k / 2, 128, 128, S128))) return rc;
    if ((rc = encode_tmap_2d_swz(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, b.codes, k / 2, b.rows, k / 2, 128, C::BNC, S128))) return rc;
    const int64_t cols = GATED ? b.rows / 2 : b.rows;
    if (OUT == DT_F32)
        rc = encode_tmap_2d_swz(&mo, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, y, cols, a.rows, cols * 4, 32, 32, S128);
    else
        rc = encode_tmap_2d_swz(&mo, OUT == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, y, cols, a.rows,
                                cols * 2, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc) return rc;
    MxParams p{};
    p.m_tiles = ceil_div(a.rows, 128 * CG);
    p.n_tiles = ceil_div(b.rows, C::BN);
    p.n = static_cast<int>(b.rows);
    p.k = k;
    p.k_chunks = kc;
    p.bias = bias;
    p.act = act;
    const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
    const int groups = (ctx->sm_count - ctx->sm_reserve) / CG;
    const int grid = static_cast<int>(tiles < groups ? tiles : groups) * CG;
    TZ_CHECK(grid > 0, TZ_EINVAL, "mxfp4 kernels need %d free SMs", CG);
    return launch_cluster(kern, CG, dim3(grid), dim3(C::THREADS), C::SMEM, s, true, ma, mb, mo, msa, msb, p, ctx->d_status);
}
// Pairs of CTAs work on 256 rows; up to 128 rows leave half of such a tile empty, so where the tiles take more than
// one round of pairs single CTAs take them (64 rows, D = 4096, 2 F = 16384: 14.8 us instead of 18.6).
template <int OUT, bool GATED>
int launch_mx(tz_ctx_t ctx, const Q4& a, const Q4& b, int k, const float* bias, void* y, int act, cudaStream_t s) {
    if (a.rows <= 128 && ceil_div(b.rows, MxCfg<1, GATED>::BN) > (ctx->sm_count - ctx->sm_reserve) / 2) return launch_mx_cg<1, OUT, GATED>(ctx, a, b, k, bias, y, act, s);
    return launch_mx_cg<kCG, OUT, GATED>(ctx, a, b, k, bias, y, act, s);
}

// The few-rows kernel, where its K slice of x fits shared memory; *ran says whether it did.
template <int N, int XDT, int OUT, bool GATED>
int launch_mx_rows(tz_ctx_t ctx, const void* x, int64_t ldx, int rows, const Q4& w, int k, const float* bias, void* y, int act, cudaStream_t s,
                   bool* ran) {
    using C = MxRowsCfg<N>;
    auto kern = mxfp4_rows_kernel<N, XDT, OUT, GATED>;
    const int tiles = ceil_div(w.rows, 128), kblocks = ceil_div(k, 256);
    *ran = false;
    if (tiles > 65535) return TZ_OK;  // the grid's second extent
    // With room for 32 rows every CTA's quantising of x weighs more, and from the third wave of CTAs on the large
    // kernel is faster: 17 / 32 rows take 22.8 / 25.2 us here and 25.3 / 25.0 there at 256 tiles (D = 4096), 28.6 / 31.3
    // and 23.1 / 22.2 us at 512 tiles (D = 2048).
    if (N > 16 && tiles > 2 * (ctx->sm_count - ctx->sm_reserve)) return TZ_OK;
    static std::atomic<unsigned> done{0};
    int rc = ensure_smem(kern, C::smem(C::MAX_KB), done);
    if (rc) return rc;
    int splits = 1;
    if ((rc = rows_splits<N * 100 + XDT * 20 + OUT * 4 + GATED + 1>(kern, C::THREADS, C::smem, ctx->sm_count - ctx->sm_reserve, tiles, kblocks, C::MAX_SPLIT, &splits)))
        return rc;
    MxRowsParams p{};
    p.kblocks = kblocks;
    p.kper = ceil_div(kblocks, splits);
    if (p.kper > C::MAX_KB) return TZ_OK;
    p.x = x;
    p.ldx = ldx;
    p.y = y;
    p.bias = bias;
    p.rows = rows;
    p.k = k;
    p.n = static_cast<int>(w.rows);
    p.k_chunks = ceil_div(k, 128);
    p.act = act;
    CUtensorMap mw, msw;
    if ((rc = encode_tmap_2d_swz(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w.codes, k / 2, w.rows, k / 2, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B)) ||
        (rc = encode_tmap_2d_swz(&msw, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, w.scales, 128, static_cast<uint64_t>(tiles) * p.k_chunks, 512, 128, 2,
                                 CU_TENSOR_MAP_SWIZZLE_NONE)))
        return rc;
    *ran = true;
    return rows_launches(ctx, tiles, splits, [&](int t0, int n, bool pdl) {
        p.tile0 = t0;
        return launch_cluster(kern, splits, dim3(splits, n), dim3(C::THREADS), C::smem(p.kper), s, pdl, mw, msw, p, ctx->d_status);
    });
}
template <int XDT, int OUT, bool GATED>
int try_mx_rows(tz_ctx_t ctx, const void* x, int64_t ldx, int64_t rows, const Q4& w, int k, const float* bias, void* y, int act, cudaStream_t s,
                bool* ran) {
    *ran = false;
    if (rows > kRowsMax) return TZ_OK;
    return rows <= 16 ? launch_mx_rows<16, XDT, OUT, GATED>(ctx, x, ldx, static_cast<int>(rows), w, k, bias, y, act, s, ran)
                      : launch_mx_rows<32, XDT, OUT, GATED>(ctx, x, ldx, static_cast<int>(rows), w, k, bias, y, act, s, ran);
}
template <int OUT>
int try_mx_rows_x(tz_ctx_t ctx, const void* x, int64_t ldx, int x_dtype, int64_t rows, const Q4& w, int k, const float* bias, void* y,
                  cudaStream_t s, bool* ran) {
    if (x_dtype == DT_F32) return try_mx_rows<DT_F32, OUT, false>(ctx, x, ldx, rows, w, k, bias, y, 0, s, ran);
    if (x_dtype == DT_F16) return try_mx_rows<DT_F16, OUT, false>(ctx, x, ldx, rows, w, k, bias, y, 0, s, ran);
    return try_mx_rows<DT_BF16, OUT, false>(ctx, x, ldx, rows, w, k, bias, y, 0, s, ran);
}

// 8 rows x 1024 columns a block.
dim3 row_grid(int64_t rows, int cols) {
    const int64_t y = (rows + 7) / 8;
    return dim3(static_cast<unsigned>(ceil_div(cols, 1024)), static_cast<unsigned>(y < 65535 ? y : 65535));
}

template <int DT, int G>
int launch_quant(tz_ctx_t ctx, const void* x, int64_t ldx, void* codes, void* scales, int64_t rows, int cols, int off, cudaStream_t s) {
    return launch_kernel(quantize_mxfp4_kernel<DT, G>, row_grid(rows, cols), dim3(256), 0, s, false, x,
                         static_cast<long long>(ldx), static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), static_cast<long long>(rows),
                         cols, off);
}
template <int G>
int quant_any(tz_ctx_t ctx, const void* x, int64_t ldx, int dtype, void* codes, void* scales, int64_t rows, int cols, int off, cudaStream_t s) {
    if (dtype == DT_F32) return launch_quant<DT_F32, G>(ctx, x, ldx, codes, scales, rows, cols, off, s);
    if (dtype == DT_F16) return launch_quant<DT_F16, G>(ctx, x, ldx, codes, scales, rows, cols, off, s);
    return launch_quant<DT_BF16, G>(ctx, x, ldx, codes, scales, rows, cols, off, s);
}

size_t a256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }
size_t code_bytes(int64_t rows, int cols) { return static_cast<size_t>(rows) * (cols / 2); }
size_t scale_bytes(int64_t rows, int cols) { return static_cast<size_t>((rows + 127) / 128) * ((cols + 127) / 128) * 512; }
size_t value_bytes(int64_t rows, int64_t cols, int dtype) { return static_cast<size_t>(rows) * cols * (dtype == DT_F32 ? 4 : 2); }
bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
Span span_of(const void* x, int64_t rows, int cols, int64_t ldx, int dtype) { return {x, rows, value_bytes(1, cols, dtype), value_bytes(1, ldx, dtype)}; }

int check_dims(const char* fn, int64_t rows, int cols) {
    TZ_CHECK(rows >= 0 && rows <= (1 << 30) && cols > 0 && cols <= (1 << 24), TZ_EINVAL, "%s: bad sizes (%lld rows, %d values)", fn,
             static_cast<long long>(rows), cols);
    TZ_CHECK(cols % 32 == 0, TZ_EINVAL, "%s: the row length must be a multiple of 32 (%d)", fn, cols);
    return TZ_OK;
}
int check_dt(const char* fn, int dtype, bool f32_ok) {
    TZ_CHECK(dtype == DT_F16 || dtype == DT_BF16 || (f32_ok && dtype == DT_F32), TZ_EINVAL, "%s: unsupported dtype %d", fn, dtype);
    return TZ_OK;
}
int check_rows(const char* fn, const void* x, int64_t ldx, int cols, int dtype) {
    const int al = dtype == DT_F32 ? 4 : 8;
    TZ_CHECK(ldx >= cols && ldx % al == 0, TZ_EINVAL, "%s: row stride %lld (at least the row length, 16-byte rows)", fn, static_cast<long long>(ldx));
    TZ_CHECK(al16(x), TZ_EINVAL, "%s: pointers must be 16-byte aligned", fn);
    return TZ_OK;
}

int product(tz_ctx_t ctx, const char* fn, const Q4& a, const Q4& w, int k, const float* bias, void* y, int y_dtype, cudaStream_t s) {
    TZ_CHECK(w.rows % 8 == 0, TZ_EINVAL, "%s: n must be a multiple of 8 (%lld)", fn, static_cast<long long>(w.rows));
    TZ_CHECK(al16(a.codes) && al16(a.scales) && al16(w.codes) && al16(w.scales) && al16(bias) && al16(y), TZ_EINVAL,
             "%s: pointers must be 16-byte aligned", fn);
    if (y_dtype == DT_F32) return launch_mx<DT_F32, false>(ctx, a, w, k, bias, y, 0, s);
    if (y_dtype == DT_F16) return launch_mx<DT_F16, false>(ctx, a, w, k, bias, y, 0, s);
    return launch_mx<DT_BF16, false>(ctx, a, w, k, bias, y, 0, s);
}

}  // namespace
}  // namespace tz

using namespace tz;

extern "C" {

int64_t tz_mxfp4_scale_bytes(int64_t rows, int cols) { return rows < 0 || cols <= 0 ? 0 : static_cast<int64_t>(scale_bytes(rows, cols)); }

int tz_quantize_mxfp4(tz_ctx_t ctx, const void* x, int64_t ldx, int dtype, void* codes, void* scales, int64_t rows, int cols, tz_stream_t stream) {
    const char* fn = "tz_quantize_mxfp4";
    TZ_CHECK(ctx, TZ_EINVAL, "%s: null context", fn);
    int rc;
    if ((rc = check_dims(fn, rows, cols)) || (rc = check_dt(fn, dtype, true))) return rc;
    if (rows == 0) return TZ_OK;
    TZ_CHECK(x && codes && scales, TZ_EINVAL, "%s: null pointer", fn);
    if ((rc = check_rows(fn, x, ldx, cols, dtype))) return rc;
    TZ_CHECK(al16(codes) && al16(scales), TZ_EINVAL, "%s: pointers must be 16-byte aligned", fn);
    const Span ix = span_of(x, rows, cols, ldx, dtype);
    if ((rc = check_apart(fn, "codes", codes, code_bytes(rows, cols), {ix})) ||
        (rc = check_apart(fn, "scales", scales, scale_bytes(rows, cols), {ix, flat(codes, code_bytes(rows, cols))})))
        return rc;
    return quant_any<0>(ctx, x, ldx, dtype, codes, scales, rows, cols, 0, pick_stream(ctx, stream));
}

int tz_dequantize_mxfp4(tz_ctx_t ctx, const void* codes, const void* scales, void* out, int dtype, int64_t rows, int cols, tz_stream_t stream) {
    const char* fn = "tz_dequantize_mxfp4";
    TZ_CHECK(ctx, TZ_EINVAL, "%s: null context", fn);
    int rc;
    if ((rc = check_dims(fn, rows, cols)) || (rc = check_dt(fn, dtype, true))) return rc;
    if (rows == 0) return TZ_OK;
    TZ_CHECK(codes && scales && out, TZ_EINVAL, "%s: null pointer", fn);
    TZ_CHECK(al16(codes) && al16(scales) && al16(out), TZ_EINVAL, "%s: pointers must be 16-byte aligned", fn);
    if ((rc = check_apart(fn, "out", out, value_bytes(rows, cols, dtype), {flat(codes, code_bytes(rows, cols)), flat(scales, scale_bytes(rows, cols))})))
        return rc;
    auto* kern = dtype == DT_F32 ? dequantize_mxfp4_kernel<DT_F32> : dtype == DT_F16 ? dequantize_mxfp4_kernel<DT_F16> : dequantize_mxfp4_kernel<DT_BF16>;
    return launch_kernel(kern, row_grid(rows, cols), dim3(256), 0, pick_stream(ctx, stream), false, static_cast<const uint8_t*>(codes),
                         static_cast<const uint8_t*>(scales), out, static_cast<long long>(rows), cols);
}

int tz_pack_gated_mxfp4(tz_ctx_t ctx, const void* w_gate, const void* w_up, int dtype, void* codes, void* scales, int f, int d, tz_stream_t stream) {
    const char* fn = "tz_pack_gated_mxfp4";
    TZ_CHECK(ctx && w_gate && w_up && codes && scales, TZ_EINVAL, "%s: null pointer", fn);
    int rc;
    if ((rc = check_dims(fn, f, d)) || (rc = check_dt(fn, dtype, true))) return rc;
    TZ_CHECK(f > 0 && f % GROUP == 0 && f <= (1 << 24), TZ_EINVAL, "%s: f must be a positive multiple of 16 (%d)", fn, f);
    if ((rc = check_rows(fn, w_gate, d, d, dtype)) || (rc = check_rows(fn, w_up, d, d, dtype))) return rc;
    TZ_CHECK(al16(codes) && al16(scales), TZ_EINVAL, "%s: pointers must be 16-byte aligned", fn);
    const Span ig = flat(w_gate, value_bytes(f, d, dtype)), iu = flat(w_up, value_bytes(f, d, dtype));
    if ((rc = check_apart(fn, "codes", codes, code_bytes(2ll * f, d), {ig, iu})) ||
        (rc = check_apart(fn, "scales", scales, scale_bytes(2ll * f, d), {ig, iu, flat(codes, code_bytes(2ll * f, d))})))
        return rc;
    cudaStream_t s = pick_stream(ctx, stream);
    if ((rc = quant_any<GROUP>(ctx, w_gate, d, dtype, codes, scales, f, d, 0, s))) return rc;
    return quant_any<GROUP>(ctx, w_up, d, dtype, codes, scales, f, d, GROUP, s);
}

int tz_gemm_mxfp4(tz_ctx_t ctx, const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales, const float* bias, void* y,
                  int y_dtype, int64_t m, int k, int n, tz_stream_t stream) {
    const char* fn = "tz_gemm_mxfp4";
    TZ_CHECK(ctx, TZ_EINVAL, "%s: null context", fn);
    int rc;
    if ((rc = check_dims(fn, m, k)) || (rc = check_dims(fn, n, k)) || (rc = check_dt(fn, y_dtype, true))) return rc;
    TZ_CHECK(n > 0, TZ_EINVAL, "%s: n must be positive", fn);
    if (m == 0) return TZ_OK;
    TZ_CHECK(a_codes && a_scales && w_codes && w_scales && y, TZ_EINVAL, "%s: null pointer", fn);
    if ((rc = check_apart(fn, "y", y, value_bytes(m, n, y_dtype),
                          {flat(a_codes, code_bytes(m, k)), flat(a_scales, scale_bytes(m, k)), flat(w_codes, code_bytes(n, k)),
                           flat(w_scales, scale_bytes(n, k)), flat(bias, bias ? 4ull * n : 0)})))
        return rc;
    return product(ctx, fn, {static_cast<const uint8_t*>(a_codes), static_cast<const uint8_t*>(a_scales), m},
                   {static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales), n}, k, bias, y, y_dtype, pick_stream(ctx, stream));
}

int tz_linear_mxfp4_workspace(int64_t m, int k, int n, size_t* bytes) {
    const char* fn = "tz_linear_mxfp4_workspace";
    TZ_CHECK(bytes, TZ_EINVAL, "%s: null argument", fn);
    int rc;
    if ((rc = check_dims(fn, m, k)) || (rc = check_dims(fn, n, k))) return rc;
    const bool in_kernel = m <= 16 && ceil_div(k, 256) <= MxRowsCfg<16>::MAX_KB && n <= 128 * 65535;  // x is quantised there
    *bytes = in_kernel ? 0 : a256(code_bytes(m, k)) + a256(scale_bytes(m, k));
    return TZ_OK;
}

// The workspace's size, and that output (`ybytes`) and workspace share no memory with the inputs or each other.
static int check_workspace(const char* fn, const void* ws, size_t ws_bytes, int64_t m, int k, int n, const Span& x, const void* w_codes,
                           const void* w_scales, const float* bias, const char* yname, const void* y, size_t ybytes) {
    size_t need = 0;
    int rc = tz_linear_mxfp4_workspace(m, k, n, &need);
    if (rc) return rc;
    TZ_CHECK(need == 0 || (ws && al16(ws) && ws_bytes >= need), TZ_EINVAL, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", fn, ws_bytes, need);
    const Span wc = flat(w_codes, code_bytes(n, k)), sc = flat(w_scales, scale_bytes(n, k)), b = flat(bias, bias ? 4ull * n : 0);
    if ((rc = check_apart(fn, yname, y, ybytes, {x, wc, sc, b}))) return rc;
    return check_apart(fn, "the workspace", ws, need, {x, wc, sc, b, flat(y, ybytes)});
}
static int quantize_input(tz_ctx_t ctx, const void* x, int64_t ldx, int x_dtype, void* ws, int64_t m, int k, cudaStream_t s, Q4* out) {
    uint8_t* codes = static_cast<uint8_t*>(ws);
    uint8_t* scales = codes + a256(code_bytes(m, k));
    *out = {codes, scales, m};
    return quant_any<0>(ctx, x, ldx, x_dtype, codes, scales, m, k, 0, s);
}

int tz_linear_mxfp4(tz_ctx_t ctx, const void* x, int64_t ldx, int x_dtype, const void* w_codes, const void* w_scales, const float* bias, void* y,
                    int y_dtype, void* workspace, size_t workspace_bytes, int64_t m, int k, int n, tz_stream_t stream) {
    const char* fn = "tz_linear_mxfp4";
    TZ_CHECK(ctx, TZ_EINVAL, "%s: null context", fn);
    int rc;
    if ((rc = check_dims(fn, m, k)) || (rc = check_dims(fn, n, k)) || (rc = check_dt(fn, x_dtype, true)) || (rc = check_dt(fn, y_dtype, true))) return rc;
    TZ_CHECK(n > 0 && n % 8 == 0, TZ_EINVAL, "%s: n must be a positive multiple of 8 (%d)", fn, n);
    if (m == 0) return TZ_OK;
    TZ_CHECK(x && w_codes && w_scales && y, TZ_EINVAL, "%s: null pointer", fn);
    if ((rc = check_rows(fn, x, ldx, k, x_dtype))) return rc;
    TZ_CHECK(al16(w_codes) && al16(w_scales) && al16(bias) && al16(y), TZ_EINVAL, "%s: pointers must be 16-byte aligned", fn);
    if ((rc = check_workspace(fn, workspace, workspace_bytes, m, k, n, span_of(x, m, k, ldx, x_dtype), w_codes, w_scales, bias, "y", y,
                              value_bytes(m, n, y_dtype))))
        return rc;
    cudaStream_t s = pick_stream(ctx, stream);
    const Q4 w{static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales), n};
    bool ran = false;
    rc = y_dtype == DT_F32   ? try_mx_rows_x<DT_F32>(ctx, x, ldx, x_dtype, m, w, k, bias, y, s, &ran)
         : y_dtype == DT_F16 ? try_mx_rows_x<DT_F16>(ctx, x, ldx, x_dtype, m, w, k, bias, y, s, &ran)
                             : try_mx_rows_x<DT_BF16>(ctx, x, ldx, x_dtype, m, w, k, bias, y, s, &ran);
    if (rc || ran) return rc;
    Q4 a;
    if ((rc = quantize_input(ctx, x, ldx, x_dtype, workspace, m, k, s, &a))) return rc;
    return product(ctx, fn, a, w, k, bias, y, y_dtype, s);
}

int tz_gated_linear_mxfp4(tz_ctx_t ctx, const void* x, int64_t ldx, int dtype, const void* w_codes, const void* w_scales, void* h, int act,
                          void* workspace, size_t workspace_bytes, int64_t t, int d, int f, tz_stream_t stream) {
    const char* fn = "tz_gated_linear_mxfp4";
    TZ_CHECK(ctx, TZ_EINVAL, "%s: null context", fn);
    int rc;
    if ((rc = check_dims(fn, t, d)) || (rc = check_dt(fn, dtype, false))) return rc;
    TZ_CHECK(gated_act_ok(act), TZ_EINVAL, "%s: activation %d is not silu, gelu, gelu_erf, relu or sigmoid", fn, act);
    TZ_CHECK(f > 0 && f % GROUP == 0 && f <= (1 << 24), TZ_EINVAL, "%s: f must be a positive multiple of 16 (%d)", fn, f);
    if (t == 0) return TZ_OK;
    TZ_CHECK(x && w_codes && w_scales && h, TZ_EINVAL, "%s: null pointer", fn);
    TZ_CHECK(al16(w_codes) && al16(w_scales) && al16(h), TZ_EINVAL, "%s: pointers must be 16-byte aligned", fn);
    if ((rc = check_rows(fn, x, ldx, d, dtype))) return rc;
    if ((rc = check_workspace(fn, workspace, workspace_bytes, t, d, 2 * f, span_of(x, t, d, ldx, dtype), w_codes, w_scales, nullptr, "h", h,
                              value_bytes(t, f, dtype))))
        return rc;
    cudaStream_t s = pick_stream(ctx, stream);
    const Q4 w{static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales), 2ll * f};
    bool ran = false;
    rc = dtype == DT_F16 ? try_mx_rows<DT_F16, DT_F16, true>(ctx, x, ldx, t, w, d, nullptr, h, act, s, &ran)
                         : try_mx_rows<DT_BF16, DT_BF16, true>(ctx, x, ldx, t, w, d, nullptr, h, act, s, &ran);
    if (rc || ran) return rc;
    Q4 a;
    if ((rc = quantize_input(ctx, x, ldx, dtype, workspace, t, d, s, &a))) return rc;
    return dtype == DT_F16 ? launch_mx<DT_F16, true>(ctx, a, w, d, nullptr, h, act, s) : launch_mx<DT_BF16, true>(ctx, a, w, d, nullptr, h, act, s);
}

}  // extern "C"
