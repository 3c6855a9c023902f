// MXFP4 (E2M1 codes, one E8M0 scale per 32 columns): the conversions shared by
// the kernels that write or read it.
//
// Scale of a block with largest magnitude a: 2^(floor(log2 a) - 2), so that
// a / scale lies in [4, 8); E2M1's largest value is 6.  Both the scale and the
// division by it are exact in f32: the biased exponent of a, less 2, is the E8M0
// code, and x / 2^(e - 127) is one multiplication by the power of two with
// exponent field 254 - e.  So codes do not depend on how a kernel splits its work.
#pragma once

#include <cuda_fp16.h>

#include "qmm_block.h"
#include "qmm_common.cuh"

namespace qmm {

constexpr int kMxBlock = 32;

__host__ __device__ constexpr int64_t mx4_pitch(int64_t k) { return (k + 31) / 32 * 16; }
// 512-byte scale tiles (128 rows x 4 blocks) along k: whole 256-column chunks.
__host__ __device__ constexpr int64_t mx4_scale_tiles(int64_t k) { return (k + 255) / 256 * 2; }
__host__ __device__ constexpr int64_t mx4_row_tiles(int64_t rows) { return (rows + 127) / 128; }

// Byte of (row, block) in the tiled scales.
__device__ __forceinline__ int64_t mx4_scale_offset(int64_t row, int64_t block, int64_t tiles) {
    return ((row >> 7) * tiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// E8M0 code from the bits of the block's largest |x| (255: infinity or NaN).
__device__ __forceinline__ uint32_t mx4_scale_code(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 1 / scale.  For code 255 the product is discarded.
__device__ __forceinline__ float mx4_inverse_scale(uint32_t code) {
    return __uint_as_float((254u - (code == 255u ? 127u : code)) << 23);
}
__device__ __forceinline__ float mx4_scale_value(uint32_t code) {
    return __uint_as_float(code == 255u ? 0x7FC00000u : code == 0u ? 0x00400000u : code << 23);
}

// Eight E2M1 codes, v[0] in the lowest four bits (round to nearest even, saturating).
__device__ __forceinline__ uint32_t mx4_pack8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The values of eight codes (exact in f16).
__device__ __forceinline__ void mx4_unpack8(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

__device__ __forceinline__ float2 mul_f32x2(float2 a, float2 b) {
    uint64_t d;
    asm("{\n\t.reg .b64 ra, rb;\n\t"
        "mov.b64 ra, {%1, %2};\n\t"
        "mov.b64 rb, {%3, %4};\n\t"
        "mul.rn.f32x2 %0, ra, rb;\n\t}\n"
        : "=l"(d)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return make_float2(__uint_as_float(static_cast<uint32_t>(d)), __uint_as_float(static_cast<uint32_t>(d >> 32)));
}
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// The larger magnitude; NaN if either is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

// Four lanes (aligned) hold a block of 32 values: the block's scale code, and
// this lane's eight codes.  Called by the whole warp.
__device__ __forceinline__ uint32_t mx4_encode8(float (&v)[8], uint32_t *codes) {
    float m = max_abs(max_abs(max_abs(v[0], v[1]), max_abs(v[2], v[3])), max_abs(max_abs(v[4], v[5]), max_abs(v[6], v[7])));
    m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t e = mx4_scale_code(__float_as_uint(m) & 0x7FFFFFFFu);
    const float2 inv = twice(mx4_inverse_scale(e));
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 t = mul_f32x2(make_float2(v[i], v[i + 1]), inv);
        v[i] = t.x;
        v[i + 1] = t.y;
    }
    const uint32_t w = mx4_pack8(v);
    *codes = e == 255u ? 0u : w;
    return e;
}

// ---------------------------------------------------------------- elements
// Typed loads and stores of the block operators (T: uint16_t tag types below
// or float).
struct Bf16 { uint16_t bits; };
struct F16 { uint16_t bits; };

__device__ __forceinline__ float elem_to_f32(Bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
__device__ __forceinline__ float elem_to_f32(F16 x) { return __half2float(__ushort_as_half(x.bits)); }
__device__ __forceinline__ float elem_to_f32(float x) { return x; }
template <typename T>
__device__ __forceinline__ T elem_from_f32(float v);
template <>
__device__ __forceinline__ Bf16 elem_from_f32<Bf16>(float v) { return Bf16{__bfloat16_as_ushort(__float2bfloat16_rn(v))}; }
template <>
__device__ __forceinline__ F16 elem_from_f32<F16>(float v) { return F16{__half_as_ushort(__float2half_rn(v))}; }
template <>
__device__ __forceinline__ float elem_from_f32<float>(float v) { return v; }

// Two 16-bit elements of a 32-bit word.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<Bf16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<F16>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<Bf16>(float a, float b) { return pack_bf16x2_rn(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<F16>(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}

// Eight consecutive elements at a 16-byte aligned address (32 bytes of f32).
template <typename T>
struct Vec8 {
    uint4 w[sizeof(T) == 4 ? 2 : 1];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load_vec8(const T *p) {
    Vec8<T> r;
    const uint4 *q = reinterpret_cast<const uint4 *>(p);
    r.w[0] = q[0];
    if constexpr (sizeof(T) == 4) r.w[1] = q[1];
    return r;
}
template <typename T>
__device__ __forceinline__ void vec8_to_f32(const Vec8<T> &r, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else {
        const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ void store_vec8(T *p, const float (&v)[8]) {
    uint4 *q = reinterpret_cast<uint4 *>(p);
    if constexpr (sizeof(T) == 4) {
        q[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        q[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
        q[0] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
}

// The same to global memory: 32 bytes of f32 in one store where the address allows, so
// that no store leaves half of a sector (B200, 16896 x 3072 codes to f32: 38 us; with
// two stores a lane 58).
template <typename T>
__device__ __forceinline__ void store_vec8_global(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        if ((reinterpret_cast<uintptr_t>(p) & 31) == 0) {
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(p)), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                         "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                         : "memory");
            return;
        }
    }
    store_vec8(p, v);
}

}  // namespace qmm
