// MXFP4 product on the tensor cores:  y [m, n] = epilogue(x [m, k] . W [n, k]^T),
// x and W in MXFP4 (qmm_mx4_linear, include/qmm_block.h).
//
// tcgen05.mma kind::mxf4 with block scaling multiplies E2M1 codes straight from
// shared memory and applies both E8M0 scales of each 32 columns inside the tensor
// core, so nothing is dequantised: products are exact and sums are f32 in tensor
// memory.  Tile: 128 tokens (A, the MMA's M) x TN features (B), 256 columns of k a
// pipeline stage = one 128-byte swizzled row per operand row (four MMAs of k = 64).
//
// The scales of 128 rows x 4 blocks are a 512-byte tile of the stored layout; the
// copy engine brings it to shared memory as it lies and one tcgen05.cp spreads it
// over the lanes of tensor memory in the form that the MMA reads (row r in lane
// r % 32 and column r / 32, four blocks a 32-bit cell, the MMA's scale id choosing
// two of them).  A feature tile of 192 starts in the middle of a 128-row scale tile
// every other time; the MMA's scale address then starts two columns in.
//
// Warp roles (one persistent CTA per SM): 8 epilogue warps (two per lane quadrant,
// each half of the columns), a producer warp (TMA for codes, bulk copies for
// scales), an MMA warp (one elected lane issues copies, MMAs and commits).  Two
// accumulators, so a tile's epilogue overlaps the next tile's main loop.  Scale
// slots in tensor memory are tied to the shared-memory stages: a stage refilled
// means that the MMAs that read its slot are complete.  Every wait is bounded.
#include <algorithm>
#include <mutex>

#include "qmm_epilogue.cuh"
#include "qmm_internal.h"
#include "qmm_mx4.cuh"

namespace qmm {
namespace mx4 {

constexpr int kTM = 128;         // tokens a tile
constexpr int kBK = 256;         // columns a stage
constexpr int kRowBytes = 128;   // codes of a row in a stage
constexpr int kSfTile = 512;     // scales of 128 rows x 4 blocks
constexpr int kEpiWarps = 8;
constexpr int kProducer = kEpiWarps, kMma = kEpiWarps + 1;
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr int kChunk = 32;       // columns an epilogue step

template <int TN>
struct Cfg {
    static_assert(TN % 64 == 0 && TN <= 256, "feature tile");
    static constexpr int kABytes = kTM * kRowBytes;
    static constexpr int kBBytes = TN * kRowBytes;
    static constexpr int kBTiles = (TN + 127) / 128;  // 128-row scale tiles under B; a start at row 64 of one still fits
    static constexpr int kSfaBytes = 2 * kSfTile;
    static constexpr int kSfbBytes = 2 * kBTiles * kSfTile;
    static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
    static constexpr int kOutBytes = kEpiWarps * 2 * kChunk * 64;  // two 32 x 32 bf16 buffers a warp
    static constexpr int kVecBytes = kEpiWarps * 2 * kChunk * 4;   // bias and gate of a chunk, a warp
    static constexpr int kSfCols = 2 * 4 * (1 + kBTiles);          // tensor-memory columns of a stage's scales
    static constexpr int kFit = (232448 - 1024 - 512 - kOutBytes - kVecBytes) / kStageBytes;
    static constexpr int kSlots = (512 - 2 * TN) / kSfCols;
    static constexpr int kStages = kFit < kSlots ? kFit : kSlots;
    static constexpr int kAOff = 0;
    static constexpr int kBOff = kAOff + kStages * kABytes;
    static constexpr int kOutOff = kBOff + kStages * kBBytes;
    static constexpr int kSfaOff = kOutOff + kOutBytes;
    static constexpr int kSfbOff = kSfaOff + kStages * kSfaBytes;
    static constexpr int kVecOff = kSfbOff + kStages * kSfbBytes;
    static constexpr int kBarOff = kVecOff + kVecBytes;
    static constexpr int kNumBars = 2 * kStages + 4 + 1 + kEpiWarps * 2;
    static constexpr int kSmemBytes = kBarOff + kNumBars * 8 + 16 + 1024;
    static constexpr int kSfCol0 = 2 * TN;
    static_assert(kStages >= 2 && kSmemBytes <= 232448, "shared memory");
    // kind::mxf4 instruction descriptor: E2M1 operands, UE8M0 scales, M = 128, N = TN.
    static constexpr uint32_t kIdesc = (1u << 7) | (1u << 10) | ((uint32_t)(TN >> 3) << 17) | (1u << 23) | ((uint32_t)(kTM >> 4) << 24);
};

struct Params {
    const uint8_t *a_scales, *b_scales;
    EpilogueArgs ep;
    uint16_t *y;
    int32_t m, n;
    int32_t nkb, sf_tiles;       // stages along k; scale tiles along k
    int32_t m_tiles, n_tiles;
    int32_t b_row_tiles;         // 128-row scale tiles of W
    int32_t tma_out;             // y (and the residual) by TMA: n % 8 == 0
    uint32_t *err;
};

// Shared-memory descriptor of a 512-byte scale tile (32 rows of 16 bytes, no
// swizzle: 8-row groups 128 bytes apart).
__device__ __forceinline__ uint64_t sdesc_scales(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(128u >> 4) << 32) | ((uint64_t)1u << 46);
}

// 32 rows x 128 bits into four tensor-memory columns, repeated in the four lane quadrants.
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void tc_mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

template <int TN>
__global__ void __launch_bounds__(kThreads, 1)
    mx4_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_y, const __grid_constant__ CUtensorMap tmap_res, const Params p) {
    using C = Cfg<TN>;
    constexpr int S = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::kBarOff);  // [S] stage landed
    uint64_t *empty = full + S;                                        // [S] stage's MMAs complete
    uint64_t *acc_full = empty + S;                                    // [2]
    uint64_t *acc_empty = acc_full + 2;                                // [2]
    uint64_t *drain = acc_empty + 2;
    uint64_t *res_full = drain + 1;                                    // [warp][2] residual chunk landed
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(res_full + kEpiWarps * 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], kEpiWarps);
        }
        mbar_init(drain, 1);
        for (int i = 0; i < kEpiWarps * 2; ++i) mbar_init(&res_full[i], 1);
        fence_barrier_init();
    }
    if (warp == kMma) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == kProducer && lane == 0) {
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
        if (p.tma_out) tma_prefetch_desc(&tmap_y);
        if (p.tma_out && p.ep.residual) tma_prefetch_desc(&tmap_res);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const int tiles = p.m_tiles * p.n_tiles;

    if (warp == kProducer) {
        // ------------------------------------------------------------ producer
        pdl_dependency_wait();
        uint32_t i = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const int m0 = t % p.m_tiles * kTM, n0 = t / p.m_tiles * TN;
            const int rt = n0 >> 7;
            const int nbt = min(C::kBTiles, p.b_row_tiles - rt);  // (TN and a start inside a tile fit kBTiles tiles)
            for (int kb = 0; kb < p.nkb; ++kb, ++i) {
                const int s = i % S;
                if (!mbar_wait(&empty[s], ((i / S) & 1) ^ 1, p.err, kErrTimeoutProducer)) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(&full[s], C::kABytes + C::kBBytes + C::kSfaBytes + nbt * 2 * kSfTile);
                    tma_load_2d(smem + C::kAOff + s * C::kABytes, &tmap_a, &full[s], kb * kRowBytes, m0);
                    tma_load_2d(smem + C::kBOff + s * C::kBBytes, &tmap_b, &full[s], kb * kRowBytes, n0);
                    bulk_load(smem + C::kSfaOff + s * C::kSfaBytes,
                              p.a_scales + ((int64_t)(m0 >> 7) * p.sf_tiles + kb * 2) * kSfTile, 2 * kSfTile, &full[s]);
                    for (int j = 0; j < nbt; ++j)
                        bulk_load(smem + C::kSfbOff + s * C::kSfbBytes + j * 2 * kSfTile,
                                  p.b_scales + ((int64_t)(rt + j) * p.sf_tiles + kb * 2) * kSfTile, 2 * kSfTile, &full[s]);
                }
                __syncwarp();
            }
        }
        pdl_launch_dependents();
        if (!ok) {  // let the copies already issued land before the CTA exits
            const uint32_t first = i > (uint32_t)S ? i - S : 0;
            for (uint32_t j = first; j < i; ++j) mbar_wait(&full[j % S], (j / S) & 1, p.err, kErrTimeoutDrain);
        }
    } else if (warp == kMma) {
        // ------------------------------------------------------------ MMA issuer
        bool ok = true, issued = false;
        uint32_t i = 0;
        int lt = 0;
        const uint64_t adesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kAOff)), bdesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kBOff));
        const uint64_t sadesc0 = sdesc_scales(smem_u32(smem + C::kSfaOff)), sbdesc0 = sdesc_scales(smem_u32(smem + C::kSfbOff));
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++lt) {
            const int n0 = t / p.m_tiles * TN;
            const int rt = n0 >> 7;
            const int nbt = min(C::kBTiles, p.b_row_tiles - rt);
            const uint32_t shift = (uint32_t)(n0 & 127) >> 5;  // columns into the first scale tile
            const int b = lt & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[b], ((lt >> 1) & 1) ^ 1, p.err, kErrTimeoutMma));
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t d = tmem + b * TN;
            uint32_t acc = 0;
            for (int kb = 0; kb < p.nkb; ++kb, ++i) {
                const uint32_t s = i % S;
                ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (i / S) & 1, p.err, kErrTimeoutMma));
                if (!ok) break;
                tc_fence_after_sync();
                if (lane_elect()) {
                    const uint32_t sfa = tmem + C::kSfCol0 + s * C::kSfCols, sfb = sfa + 8;
                    const uint64_t ad = adesc0 + (uint64_t)s * (C::kABytes >> 4), bd = bdesc0 + (uint64_t)s * (C::kBBytes >> 4);
                    const uint64_t sad = sadesc0 + (uint64_t)s * (C::kSfaBytes >> 4), sbd = sbdesc0 + (uint64_t)s * (C::kSfbBytes >> 4);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // 128 columns: one scale tile along k
                        tc_copy_scales(sfa + h * 4, sad + h * (kSfTile >> 4));
                        for (int j = 0; j < nbt; ++j)
                            tc_copy_scales(sfb + h * 4 * C::kBTiles + j * 4, sbd + (j * 2 + h) * (kSfTile >> 4));
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint32_t id = (kk & 1) * 2;  // which two of the cell's four scales
                        tc_mma_mxf4(d, ad + kk * 2, bd + kk * 2, C::kIdesc | (id << 4) | (id << 29), sfa + (kk >> 1) * 4,
                                    sfb + (kk >> 1) * 4 * C::kBTiles + shift, acc);
                        acc = 1;
                    }
                    tc_commit(&empty[s]);
                }
                issued = true;
            }
            if (!ok) break;
            if (lane_elect()) tc_commit(&acc_full[b]);
            __syncwarp();
        }
        if (!ok && issued) {
            if (lane_elect()) tc_commit(drain);
            __syncwarp();
            mbar_wait(drain, 0, p.err, kErrTimeoutDrain);
        }
    } else {
        // ------------------------------------------------------------ epilogue
        pdl_dependency_wait();
        const int quad = warp & 3, half = warp >> 2;
        constexpr int kChunks = TN / 2 / kChunk;  // chunks of this warp's half
        uint8_t *const out = smem + C::kOutOff + warp * 2 * kChunk * 64;
        float *const vec = reinterpret_cast<float *>(smem + C::kVecOff) + warp * 2 * kChunk;
        uint64_t *const rbar = res_full + warp * 2;
        const bool res_tma = p.tma_out && p.ep.residual;
        uint32_t q = 0;  // chunks so far
        int lt = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++lt) {
            const int m0 = t % p.m_tiles * kTM + quad * 32, n0 = t / p.m_tiles * TN + half * (TN / 2);
            const int row = m0 + lane;
            const int b = lt & 1;
            // A quadrant past the last token or a chunk past the last feature has nothing to store.
            const int chunks = m0 < p.m ? min(kChunks, (p.n - n0 + kChunk - 1) / kChunk) : 0;
            auto load_residual = [&](int c, uint32_t buf) {
                if (lane == 0) {
                    bulk_wait_read<0>();  // stores from this buffer have left it
                    mbar_arrive_expect_tx(&rbar[buf], kChunk * 64);
                    tma_load_2d(out + buf * kChunk * 64, &tmap_res, &rbar[buf], n0 + c * kChunk, m0);
                }
            };
            if (res_tma && chunks > 0) load_residual(0, q & 1);
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (lt >> 1) & 1, p.err, kErrTimeoutEpilogue))) {
                if (res_tma && chunks > 0) mbar_wait(&rbar[q & 1], (q >> 1) & 1, p.err, kErrTimeoutDrain);
                break;
            }
            tc_fence_after_sync();
            bool ok = true;
            for (int c = 0; c < chunks; ++c, ++q) {
                const uint32_t buf = q & 1;
                uint8_t *const o = out + buf * kChunk * 64;
                const int f0 = n0 + c * kChunk;
                uint32_t r[32];
                tmem_ld_32x32b_x32(tmem + ((uint32_t)(quad * 32) << 16) + b * TN + half * (TN / 2) + c * kChunk, r);
                if (res_tma) {
                    if (c + 1 < chunks) load_residual(c + 1, buf ^ 1);
                } else if (lane == 0) {
                    bulk_wait_read<1>();
                }
                {
                    const FeatureConsts fc = load_feature_consts(p.ep, f0 + lane, f0 + lane < p.n);
                    __syncwarp();
                    vec[lane] = fc.bias;
                    vec[kChunk + lane] = fc.gate;
                    __syncwarp();
                }
                if (res_tma) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&rbar[buf], (q >> 1) & 1, p.err, kErrTimeoutEpilogue));
                    if (!ok) {
                        if (c + 1 < chunks) mbar_wait(&rbar[buf ^ 1], ((q + 1) >> 1) & 1, p.err, kErrTimeoutDrain);
                        break;
                    }
                }
                tc_wait_ld();
#pragma unroll
                for (int g = 0; g < 4; ++g) {  // eight features: 16 bytes of this token's row
                    uint4 *const cell = reinterpret_cast<uint4 *>(o + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4));
                    float v[8], res[8];
                    if (p.ep.residual) {
                        if (res_tma) {
                            Vec8<Bf16> w;
                            w.w[0] = *cell;
                            vec8_to_f32(w, res);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int f = f0 + g * 8 + e;
                                res[e] = row < p.m && f < p.n ? bf16_bits_to_f32(p.ep.residual[(int64_t)row * p.n + f]) : 0.0f;
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const FeatureConsts fc{vec[g * 8 + e], vec[kChunk + g * 8 + e]};
                        v[e] = epilogue_value_rv(p.ep, fc, __uint_as_float(r[g * 8 + e]), p.ep.residual ? res[e] : 0.0f);
                    }
                    *cell = make_uint4(pack_bf16x2_rn(v[0], v[1]), pack_bf16x2_rn(v[2], v[3]), pack_bf16x2_rn(v[4], v[5]),
                                       pack_bf16x2_rn(v[6], v[7]));
                }
                if (p.tma_out) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmap_y, o, f0, m0);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    const int rows = min(32, p.m - m0);
                    for (int rr = 0; rr < rows; ++rr) {
                        const uint16_t v = *reinterpret_cast<const uint16_t *>(o + rr * 64 + (((lane >> 3) ^ ((rr >> 1) & 3)) << 4) + (lane & 7) * 2);
                        if (f0 + lane < p.n) p.y[(int64_t)(m0 + rr) * p.n + f0 + lane] = v;
                    }
                }
                __syncwarp();
            }
            if (!ok) break;
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
        }
        if (lane == 0) bulk_wait_all();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kMma) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                   const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    });
    return fn;
}

static qmm_status map_2d(CUtensorMap *map, CUtensorMapDataType type, const void *base, uint64_t inner, uint64_t outer, uint64_t row_bytes,
                         uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle swz) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(QMM_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[2] = {inner, outer};
    cuuint64_t strides[1] = {row_bytes};
    cuuint32_t box[2] = {box_inner, box_outer};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, type, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(QMM_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return QMM_OK;
}

template <int TN>
static qmm_status launch_gemm(const qmm_mx4 &w, const qmm_mx4 &x, const qmm_epilogue &ep, uint16_t *y, cudaStream_t st) {
    using C = Cfg<TN>;
    auto kernel = mx4_gemm_kernel<TN>;
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return cuda_fail(e, "mxfp4 gemm smem attribute");
        configured[dev] = true;
    }
    const uint64_t pitch = (uint64_t)mx4_pitch(w.k);
    CUtensorMap ta, tb, ty, tr;
    qmm_status s = map_2d(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, x.codes, pitch, (uint64_t)x.rows, pitch, kRowBytes, kTM, CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != QMM_OK) return s;
    s = map_2d(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes, pitch, (uint64_t)w.rows, pitch, kRowBytes, TN, CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != QMM_OK) return s;
    const bool tma_out = w.rows % 8 == 0;  // rows of y on 16-byte boundaries
    ty = tr = ta;
    if (tma_out) {
        s = map_2d(&ty, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, y, (uint64_t)w.rows, (uint64_t)x.rows, (uint64_t)w.rows * 2, kChunk, 32, CU_TENSOR_MAP_SWIZZLE_64B);
        if (s == QMM_OK && ep.residual)
            s = map_2d(&tr, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ep.residual, (uint64_t)w.rows, (uint64_t)x.rows, (uint64_t)w.rows * 2, kChunk, 32,
                       CU_TENSOR_MAP_SWIZZLE_64B);
        if (s != QMM_OK) return s;
    }
    Params p;
    p.a_scales = x.scales;
    p.b_scales = w.scales;
    p.ep = epilogue_args(ep);
    p.y = y;
    p.m = (int32_t)x.rows;
    p.n = (int32_t)w.rows;
    p.nkb = (int32_t)((w.k + kBK - 1) / kBK);
    p.sf_tiles = (int32_t)mx4_scale_tiles(w.k);
    p.m_tiles = (int32_t)((x.rows + kTM - 1) / kTM);
    p.n_tiles = (int32_t)((w.rows + TN - 1) / TN);
    p.b_row_tiles = (int32_t)mx4_row_tiles(w.rows);
    p.tma_out = tma_out ? 1 : 0;
    p.err = device_error_word();
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    if (tiles > INT32_MAX / 2) return fail(QMM_ERR_UNSUPPORTED, "mxfp4 linear: too many output tiles");
    const unsigned grid = (unsigned)std::min<int64_t>(tiles, sm_count());
    kernel<<<grid, kThreads, C::kSmemBytes, st>>>(ta, tb, ty, tr, p);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? QMM_OK : cuda_fail(e, "mxfp4 gemm launch");
}

}  // namespace mx4
}  // namespace qmm

using qmm::fail;

namespace {

struct Span {
    uintptr_t lo, hi;
};
Span span(const void *p, uint64_t bytes) {
    return Span{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + (uintptr_t)bytes};
}
bool overlap(const Span &a, const Span &b) { return a.lo < b.hi && b.lo < a.hi; }
bool misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
uint64_t round16(uint64_t v) { return (v + 15) / 16 * 16; }

}  // namespace

extern "C" {

uint64_t qmm_mx4_workspace_bytes(int64_t m, int64_t k) {
    return round16(qmm_mx4_code_bytes(m, k)) + qmm_mx4_scale_bytes(m, k);
}

qmm_status qmm_mx4_linear(const qmm_mx4_linear_args *p, void *stream) {
    if (!p) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: null arguments");
    const qmm_mx4_linear_args &a = *p;
    if (a.m < 0 || a.w.rows <= 0 || a.w.k <= 0)
        return fail(QMM_ERR_BAD_SHAPE, "mxfp4 linear: %lld tokens, %lldx%lld weight", (long long)a.m, (long long)a.w.rows, (long long)a.w.k);
    if (a.m > INT32_MAX - 256 || a.w.rows > INT32_MAX - 256 || a.w.k > INT32_MAX / 4)
        return fail(QMM_ERR_UNSUPPORTED, "mxfp4 linear: %lld tokens, %lldx%lld weight are past the kernel's indexes", (long long)a.m, (long long)a.w.rows, (long long)a.w.k);
    const int32_t act = a.activation & 0xFF;
    if ((a.activation & ~(0xFF | QMM_EPILOGUE_RESIDUAL_MUL)) != 0 || act < QMM_ACT_NONE || act > QMM_ACT_SILU)
        return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: unknown activation %d", a.activation);
    const bool quantised = a.x_codes || a.x_scales;
    if (a.m == 0) return QMM_OK;
    if (!a.w.codes || !a.w.scales || !a.y) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: null weight or y");
    if (quantised ? (!a.x_codes || !a.x_scales || a.x != nullptr) : !a.x)
        return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: x is either a matrix or codes with scales");
    if (!quantised && (a.x_elem < QMM_ELEM_BF16 || a.x_elem > QMM_ELEM_F16)) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: element type %d", a.x_elem);
    if (!quantised && a.m > 1 && a.x_row_stride < a.w.k)
        return fail(QMM_ERR_BAD_SHAPE, "mxfp4 linear: row stride %lld below %lld columns", (long long)a.x_row_stride, (long long)a.w.k);
    if (misaligned(a.w.codes) || misaligned(a.w.scales) || misaligned(a.y) || misaligned(a.residual) || misaligned(a.x_codes) || misaligned(a.x_scales))
        return fail(QMM_ERR_MISALIGNED, "mxfp4 linear: codes, scales, y and residual must be 16-byte aligned");
    const uintptr_t xsize = a.x_elem == QMM_ELEM_F32 ? 4 : 2;
    if ((!quantised && reinterpret_cast<uintptr_t>(a.x) % xsize) || ((reinterpret_cast<uintptr_t>(a.bias) | reinterpret_cast<uintptr_t>(a.gate)) & 1))
        return fail(QMM_ERR_MISALIGNED, "mxfp4 linear: x, bias or gate is not aligned to its element");
    const uint64_t code_bytes = qmm_mx4_code_bytes(a.m, a.w.k), scale_bytes = qmm_mx4_scale_bytes(a.m, a.w.k);
    const Span sy = span(a.y, (uint64_t)a.m * (uint64_t)a.w.rows * 2);
    const Span sw[] = {span(a.w.codes, qmm_mx4_code_bytes(a.w.rows, a.w.k)), span(a.w.scales, qmm_mx4_scale_bytes(a.w.rows, a.w.k))};
    Span sx[] = {span(a.x_codes, quantised ? code_bytes : 0), span(a.x_scales, quantised ? scale_bytes : 0)};
    qmm_mx4 x{a.x_codes, a.x_scales, a.m, a.w.k};
    if (!quantised) {
        const uint64_t need = qmm_mx4_workspace_bytes(a.m, a.w.k);
        if (!a.workspace || a.workspace_bytes < need)
            return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: workspace of %llu bytes is smaller than %llu", (unsigned long long)a.workspace_bytes, (unsigned long long)need);
        if (misaligned(a.workspace)) return fail(QMM_ERR_MISALIGNED, "mxfp4 linear: workspace is not 16-byte aligned");
        sx[0] = span(a.x, ((uint64_t)(a.m - 1) * (uint64_t)a.x_row_stride + (uint64_t)a.w.k) * xsize);
        sx[1] = span(a.workspace, need);
        if (overlap(sx[0], sx[1]) || overlap(sx[1], sw[0]) || overlap(sx[1], sw[1]) ||
            (a.residual && overlap(sx[1], span(a.residual, (uint64_t)a.m * (uint64_t)a.w.rows * 2))))
            return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: workspace overlaps an operand");
        x.codes = static_cast<uint8_t *>(a.workspace);
        x.scales = x.codes + round16(code_bytes);
    }
    if (overlap(sy, sx[0]) || overlap(sy, sx[1]) || overlap(sy, sw[0]) || overlap(sy, sw[1]))
        return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: y overlaps x, the weight or the workspace");
    if (a.residual && a.residual != a.y && overlap(sy, span(a.residual, (uint64_t)a.m * (uint64_t)a.w.rows * 2)))
        return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: the residual overlaps y without being it");
    qmm_status s = qmm::check_device();
    if (s != QMM_OK) return s;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!quantised) {
        s = qmm::launch_mx4_quantize(a.x, a.x_elem, a.m, a.w.k, a.x_row_stride, const_cast<uint8_t *>(x.codes), const_cast<uint8_t *>(x.scales), st);
        if (s != QMM_OK) return s;
    }
    const qmm_epilogue ep{a.bias, a.gate, a.residual, a.activation};
    return qmm::mx4::launch_gemm<192>(a.w, x, ep, a.y, st);
}

}  // extern "C"
