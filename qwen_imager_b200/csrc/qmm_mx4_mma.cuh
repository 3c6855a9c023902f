// What the MXFP4 product kernels share: scale copies and block-scaled MMAs, the
// epilogue's activations, tensor maps.
#pragma once

#include <mutex>

#include "qmm_epilogue.cuh"
#include "qmm_internal.h"
#include "qmm_mx4.cuh"

namespace qmm {
namespace mx4 {

constexpr int kBK = 256;        // columns a stage: a 128-byte swizzled row of codes, four MMAs of k = 64
constexpr int kRowBytes = 128;
constexpr int kSfTile = 512;    // scales of 128 rows x 4 blocks

// kind::mxf4 instruction descriptor: E2M1 operands, both K-major, UE8M0 scales, f32 accumulators.
__host__ __device__ constexpr uint32_t idesc_mxf4(uint32_t m, uint32_t n) {
    return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24);
}
// Which two of a 32-bit cell's four scales the MMA takes, for both operands: 0 or 2.
__device__ __forceinline__ uint32_t idesc_scale_id(uint32_t id) { return (id << 4) | (id << 29); }

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

// t * sigmoid(z) of two values: both activations in one exponential and one
// reciprocal a value (GELU's 0.5 (1 + tanh u) is sigmoid(2 u)).  Beside a few 2^-22 of
// the fast forms, the rounding of the exponent y = -z log2(e) costs about |y| 2^-23 of
// the result where t is negative: 2^-16 at the most, as past |y| = 126 (results below
// 1e-36) it is 0; the rounding to bf16 is 2^-8.  Past their range the forms give 0 or t.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool GELU>
__device__ __forceinline__ float2 activate(float2 t) {
    const float2 zero = make_float2(0.0f, 0.0f);
    constexpr float kLog2e = 1.4426950408889634f, kGelu = 1.5957691216057308f;  // 2 sqrt(2 / pi)
    float2 z;  // -z log2(e)
    if constexpr (GELU) {
        const float2 a = make_float2(-kGelu * kLog2e, -kGelu * kLog2e), b = make_float2(-kGelu * kLog2e * 0.044715f, -kGelu * kLog2e * 0.044715f);
        z = fma_f32x2(fma_f32x2(fma_f32x2(t, t, zero), b, a), t, zero);
    } else {
        z = fma_f32x2(t, make_float2(-kLog2e, -kLog2e), zero);
    }
    const float2 d = add_f32x2(make_float2(exp2_fast(z.x), exp2_fast(z.y)), make_float2(1.0f, 1.0f));
    return make_float2(t.x * rcp_fast(d.x), t.y * rcp_fast(d.y));
}

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                   const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
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

inline qmm_status map_2d(CUtensorMap *map, CUtensorMapDataType type, const void *base, uint64_t inner, uint64_t outer, uint64_t row_bytes,
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

template <typename K>
inline qmm_status allow_smem(K kernel, int bytes, bool (&configured)[64]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return cuda_fail(e, "mxfp4 gemm smem attribute");
        configured[dev] = true;
    }
    return QMM_OK;
}

// The product for few tokens (qmm_mx4_small.cu): whether it is the kernel for [m, k] .
// [n, k]^T, whether it then quantises x itself, and its launch (x null: xq holds x).
bool mx4_small_fits(int64_t n, int64_t m);
bool mx4_small_quantises(int64_t n, int64_t m, int64_t k);
qmm_status launch_mx4_small(const qmm_mx4 &w, const void *x, int32_t elem, int64_t x_row_stride, const qmm_mx4 &xq, const qmm_epilogue &ep,
                            uint16_t *y, cudaStream_t st);

}  // namespace mx4
}  // namespace qmm
