// MXFP4 quantisation, its inverse, and the order of the scales
// (include/qmm_block.h).
//
// HBM-bound: quantisation reads x once and writes 17 bytes per 32 columns,
// dequantisation the reverse.  One warp takes a chunk of 256 columns (eight per
// lane, four lanes a block) of the four rows i, i + 32, i + 64, i + 96 of a
// 128-row scale tile: the four rows' scales of four blocks are 16 consecutive
// bytes of the tile, so they leave in one store, and the four rows' loads are in
// flight together.  Rows that are not 16-byte aligned pass through a per-warp
// shared buffer, so that global accesses stay consecutive across the lanes.
// B200, 16896 x 3072 bf16: quantised and back in 45 us (264 MB: 0.90 of the measured HBM
// rate), 25 and 21 us each; 1153 x 4307 f32, unaligned, 10 us (two launches of 4 us).
#include "qmm_internal.h"
#include "qmm_mx4.cuh"

namespace qmm {
namespace mx4 {

constexpr int kWarps = 8;
constexpr int kRows = 4;  // rows of a tile per warp

struct QuantArgs {
    const void *x;
    int64_t rows, k, row_stride;
    uint8_t *codes, *scales;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) quantize_kernel(const QuantArgs a) {
    __shared__ __align__(16) T stage[VEC ? 1 : kWarps][VEC ? 8 : 256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = (blockIdx.y & 3) * kWarps + warp;  // row within 32
    const int64_t row0 = (int64_t)(blockIdx.y >> 2) * 128 + i;
    const int64_t col0 = (int64_t)blockIdx.x * 256;
    const T *x = static_cast<const T *>(a.x);
    pdl_launch_dependents();  // a product behind this pass sets itself up meanwhile; it waits for the grid before it reads
    if (row0 >= a.rows) return;
    float v[kRows][8];
    if constexpr (VEC) {  // k is a multiple of 8: a lane's columns are all in or all out
        Vec8<T> raw[kRows];
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            raw[j] = Vec8<T>{};
            const int64_t r = row0 + 32 * j, c = col0 + lane * 8;
            if (r < a.rows && c < a.k) raw[j] = load_vec8(x + r * a.row_stride + c);
        }
#pragma unroll
        for (int j = 0; j < kRows; ++j) vec8_to_f32(raw[j], v[j]);
    } else {
        T e[kRows][8];
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int64_t r = row0 + 32 * j;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int64_t c = col0 + q * 32 + lane;
                e[j][q] = T{};
                if (r < a.rows && c < a.k) e[j][q] = x[r * a.row_stride + c];
            }
        }
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 8; ++q) stage[warp][q * 32 + lane] = e[j][q];
            __syncwarp();
            vec8_to_f32(load_vec8(&stage[warp][lane * 8]), v[j]);
        }
    }
    const int64_t pitch = mx4_pitch(a.k);
    uint32_t sc[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        uint32_t w;
        const uint32_t e = mx4_encode8(v[j], &w);
        const int64_t r = row0 + 32 * j, byte = (int64_t)blockIdx.x * 128 + lane * 4;
        if (r < a.rows && byte < pitch) *reinterpret_cast<uint32_t *>(a.codes + r * pitch + byte) = w;
        // the four blocks of this half of the warp in one word
        uint32_t word = e << (8 * ((lane >> 2) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        sc[j] = word;
    }
    if ((lane & 15) == 0) {
        const int64_t tile = (int64_t)(blockIdx.y >> 2) * mx4_scale_tiles(a.k) + blockIdx.x * 2 + (lane >> 4);
        *reinterpret_cast<uint4 *>(a.scales + tile * 512 + i * 16) = make_uint4(sc[0], sc[1], sc[2], sc[3]);
    }
}

struct DequantArgs {
    const uint8_t *codes, *scales;
    int64_t rows, k;
    void *dst;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const DequantArgs a) {
    __shared__ __align__(16) T stage[VEC ? 1 : kWarps][VEC ? 8 : 256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = (blockIdx.y & 3) * kWarps + warp;
    const int64_t row0 = (int64_t)(blockIdx.y >> 2) * 128 + i;
    const int64_t col0 = (int64_t)blockIdx.x * 256;
    T *dst = static_cast<T *>(a.dst);
    if (row0 >= a.rows) return;
    const int64_t pitch = mx4_pitch(a.k);
    const int64_t tile = (int64_t)(blockIdx.y >> 2) * mx4_scale_tiles(a.k) + blockIdx.x * 2 + (lane >> 4);
    const uint4 s4 = __ldg(reinterpret_cast<const uint4 *>(a.scales + tile * 512 + i * 16));
    const uint32_t sw[4] = {s4.x, s4.y, s4.z, s4.w};
    uint32_t w[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const int64_t r = row0 + 32 * j, byte = (int64_t)blockIdx.x * 128 + lane * 4;
        w[j] = 0;
        if (r < a.rows && byte < pitch) w[j] = __ldg(reinterpret_cast<const uint32_t *>(a.codes + r * pitch + byte));
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
        const int64_t r = row0 + 32 * j;
        if (r >= a.rows) break;
        float v[8];
        mx4_unpack8(w[j], v);
        const float s = mx4_scale_value((sw[j] >> (8 * ((lane >> 2) & 3))) & 255u);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] *= s;
        if constexpr (VEC) {
            const int64_t c = col0 + lane * 8;
            if (c < a.k) store_vec8_global(dst + r * a.k + c, v);
        } else {
            __syncwarp();
            store_vec8(&stage[warp][lane * 8], v);
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int64_t c = col0 + q * 32 + lane;
                if (c < a.k) dst[r * a.k + c] = stage[warp][q * 32 + lane];
            }
        }
    }
}

// Row-major <-> tiled scales, a thread per byte.
template <bool TILE>
__global__ void scale_order_kernel(const uint8_t *__restrict__ src, uint8_t *__restrict__ dst, int64_t rows, int64_t blocks,
                                   int64_t tiles) {
    const int64_t padded = tiles * 4;
    const int64_t total = rows * (TILE ? padded : blocks);
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / (TILE ? padded : blocks), b = i % (TILE ? padded : blocks);
        if constexpr (TILE) dst[mx4_scale_offset(r, b, tiles)] = b < blocks ? src[r * blocks + b] : 0;
        else dst[r * blocks + b] = src[mx4_scale_offset(r, b, tiles)];
    }
}

// Grid of 256-column chunks x (row tiles x 4 groups of 8 rows); false when it is past the launch limits.
static bool chunk_grid(int64_t rows, int64_t k, dim3 *grid) {
    const int64_t x = (k + 255) / 256, y = mx4_row_tiles(rows) * 4;
    if (x > INT32_MAX || y > 65535) return false;
    *grid = dim3((unsigned)x, (unsigned)y, 1);
    return true;
}

template <typename T>
static void launch_quantize(const dim3 &grid, const QuantArgs &a, cudaStream_t st) {
    const bool vec = a.k % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (a.row_stride * (int64_t)sizeof(T)) % 16 == 0;
    if (vec) quantize_kernel<T, true><<<grid, kWarps * 32, 0, st>>>(a);
    else quantize_kernel<T, false><<<grid, kWarps * 32, 0, st>>>(a);
}

template <typename T>
static void launch_dequantize(const dim3 &grid, const DequantArgs &a, cudaStream_t st) {
    if (a.k % 8 == 0 && (reinterpret_cast<uintptr_t>(a.dst) & 15) == 0) dequantize_kernel<T, true><<<grid, kWarps * 32, 0, st>>>(a);
    else dequantize_kernel<T, false><<<grid, kWarps * 32, 0, st>>>(a);
}

// Rows per launch: the grid's y extent holds 65535 / 4 row tiles.
constexpr int64_t kRowsPerLaunch = 65535 / 4 * 128;

}  // namespace mx4

qmm_status launch_mx4_quantize(const void *x, int32_t elem, int64_t rows, int64_t k, int64_t row_stride, uint8_t *codes,
                               uint8_t *scales, cudaStream_t st) {
    const int64_t esize = elem == QMM_ELEM_F32 ? 4 : 2;
    for (int64_t r = 0; r < rows; r += mx4::kRowsPerLaunch) {
        const mx4::QuantArgs a{static_cast<const uint8_t *>(x) + r * row_stride * esize,
                               rows - r < mx4::kRowsPerLaunch ? rows - r : mx4::kRowsPerLaunch, k, row_stride,
                               codes + r * mx4_pitch(k), scales + r / 128 * mx4_scale_tiles(k) * 512};
        dim3 grid;
        if (!mx4::chunk_grid(a.rows, k, &grid)) return fail(QMM_ERR_UNSUPPORTED, "mxfp4: %lld columns are past the launch limits", (long long)k);
        if (elem == QMM_ELEM_F32) mx4::launch_quantize<float>(grid, a, st);
        else if (elem == QMM_ELEM_F16) mx4::launch_quantize<F16>(grid, a, st);
        else mx4::launch_quantize<Bf16>(grid, a, st);
        count_launch();
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "mxfp4 quantize launch");
    }
    return QMM_OK;
}

static qmm_status check_shape(const char *what, int64_t rows, int64_t k) {
    if (rows < 0 || k <= 0 || k > INT32_MAX || rows > INT64_MAX / 8 / (k + 256))
        return fail(QMM_ERR_BAD_SHAPE, "%s: %lld rows of %lld", what, (long long)rows, (long long)k);
    return QMM_OK;
}

static bool misaligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace qmm

using qmm::fail;

extern "C" {

uint64_t qmm_mx4_code_bytes(int64_t rows, int64_t k) {
    return rows <= 0 || k <= 0 ? 0 : (uint64_t)rows * (uint64_t)qmm::mx4_pitch(k);
}

uint64_t qmm_mx4_scale_bytes(int64_t rows, int64_t k) {
    return rows <= 0 || k <= 0 ? 0 : (uint64_t)qmm::mx4_row_tiles(rows) * (uint64_t)qmm::mx4_scale_tiles(k) * 512u;
}

qmm_status qmm_mx4_quantize(const void *x, int32_t elem, int64_t rows, int64_t k, int64_t row_stride, uint8_t *codes,
                            uint8_t *scales, void *stream) {
    qmm_status s = qmm::check_shape("mxfp4 quantize", rows, k);
    if (s != QMM_OK) return s;
    if (elem < QMM_ELEM_BF16 || elem > QMM_ELEM_F16) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 quantize: element type %d", elem);
    if (rows == 0) return QMM_OK;
    if (!x || !codes || !scales) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 quantize: null pointer");
    if (row_stride < k && rows > 1) return fail(QMM_ERR_BAD_SHAPE, "mxfp4 quantize: row stride %lld below %lld columns", (long long)row_stride, (long long)k);
    if (qmm::misaligned(codes) || qmm::misaligned(scales)) return fail(QMM_ERR_MISALIGNED, "mxfp4 quantize: codes and scales must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(x) % (elem == QMM_ELEM_F32 ? 4 : 2)) return fail(QMM_ERR_MISALIGNED, "mxfp4 quantize: x is not aligned to its element");
    if ((s = qmm::check_device()) != QMM_OK) return s;
    return qmm::launch_mx4_quantize(x, elem, rows, k, row_stride, codes, scales, static_cast<cudaStream_t>(stream));
}

qmm_status qmm_mx4_dequantize(const qmm_mx4 *w, void *dst, int32_t elem, void *stream) {
    if (!w) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 dequantize: null matrix");
    qmm_status s = qmm::check_shape("mxfp4 dequantize", w->rows, w->k);
    if (s != QMM_OK) return s;
    if (elem < QMM_ELEM_BF16 || elem > QMM_ELEM_F16) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 dequantize: element type %d", elem);
    if (w->rows == 0) return QMM_OK;
    if (!w->codes || !w->scales || !dst) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 dequantize: null pointer");
    if (qmm::misaligned(w->codes) || qmm::misaligned(w->scales)) return fail(QMM_ERR_MISALIGNED, "mxfp4 dequantize: codes and scales must be 16-byte aligned");
    const int64_t esize = elem == QMM_ELEM_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(dst) % esize) return fail(QMM_ERR_MISALIGNED, "mxfp4 dequantize: dst is not aligned to its element");
    if ((s = qmm::check_device()) != QMM_OK) return s;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (int64_t r = 0; r < w->rows; r += qmm::mx4::kRowsPerLaunch) {
        const qmm::mx4::DequantArgs a{w->codes + r * qmm::mx4_pitch(w->k), w->scales + r / 128 * qmm::mx4_scale_tiles(w->k) * 512,
                                      w->rows - r < qmm::mx4::kRowsPerLaunch ? w->rows - r : qmm::mx4::kRowsPerLaunch, w->k,
                                      static_cast<uint8_t *>(dst) + r * w->k * esize};
        dim3 grid;
        if (!qmm::mx4::chunk_grid(a.rows, a.k, &grid)) return fail(QMM_ERR_UNSUPPORTED, "mxfp4: %lld columns are past the launch limits", (long long)a.k);
        if (elem == QMM_ELEM_F32) qmm::mx4::launch_dequantize<float>(grid, a, st);
        else if (elem == QMM_ELEM_F16) qmm::mx4::launch_dequantize<qmm::F16>(grid, a, st);
        else qmm::mx4::launch_dequantize<qmm::Bf16>(grid, a, st);
        qmm::count_launch();
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return qmm::cuda_fail(e, "mxfp4 dequantize launch");
    }
    return QMM_OK;
}

static qmm_status scale_order(bool tile, const uint8_t *src, int64_t rows, int64_t k, uint8_t *dst, void *stream) {
    qmm_status s = qmm::check_shape("mxfp4 scales", rows, k);
    if (s != QMM_OK) return s;
    if (rows == 0) return QMM_OK;
    if (!src || !dst) return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 scales: null pointer");
    if ((s = qmm::check_device()) != QMM_OK) return s;
    const int64_t blocks = (k + 31) / 32, tiles = qmm::mx4_scale_tiles(k);
    const int64_t work = rows * (tile ? tiles * 4 : blocks);
    const unsigned grid = (unsigned)(work / 256 + 1 < 4736 ? work / 256 + 1 : 4736);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (tile) qmm::mx4::scale_order_kernel<true><<<grid, 256, 0, st>>>(src, dst, rows, blocks, tiles);
    else qmm::mx4::scale_order_kernel<false><<<grid, 256, 0, st>>>(src, dst, rows, blocks, tiles);
    qmm::count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? QMM_OK : qmm::cuda_fail(e, "mxfp4 scale order launch");
}

qmm_status qmm_mx4_tile_scales(const uint8_t *row_major, int64_t rows, int64_t k, uint8_t *scales, void *stream) {
    return scale_order(true, row_major, rows, k, scales, stream);
}

qmm_status qmm_mx4_row_scales(const uint8_t *scales, int64_t rows, int64_t k, uint8_t *row_major, void *stream) {
    return scale_order(false, scales, rows, k, row_major, stream);
}

}  // extern "C"
