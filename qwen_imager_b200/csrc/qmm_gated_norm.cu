// The seam between two sublayers of a block (qmm_gated_residual_norm):
//   h  = norm_post(branch) * post_weight
//   x' = residual_scale * x + gate * h
//   n  = norm_pre(x') * pre_weight * (1 + scale) + shift
// HBM-bound: x and branch are read once, x' and n (or its MXFP4 codes) written
// once.  One CTA per row: the row stays in registers (eight columns a vector, one
// to four vectors a thread), so mean and variance are two passes over registers,
// and each statistic costs one shuffle tree, one shared slot a warp and one
// barrier.  All loads of the row are issued before the first reduction.
// Rows that are not 16-byte aligned use the same kernel with columns dealt out
// one by one (thread t holds columns t, t + T, ...), which keeps accesses of a
// warp consecutive.
#include "qmm_internal.h"
#include "qmm_mx4.cuh"

namespace qmm {
namespace gnorm {

// Eight elements of a runtime type at an aligned address, kept raw until used.
struct Raw8 {
    uint4 a, b;
};
__device__ __forceinline__ Raw8 load_raw8(const void *p, int elem, int64_t index) {
    Raw8 r{};
    if (elem == QMM_ELEM_F32) {
        const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + index);
        r.a = q[0];
        r.b = q[1];
    } else {
        r.a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + index);
    }
    return r;
}
__device__ __forceinline__ void raw8_to_f32(const Raw8 &r, int elem, float (&v)[8]) {
    if (elem == QMM_ELEM_F32) {
        Vec8<float> t;
        t.w[0] = r.a;
        t.w[1] = r.b;
        vec8_to_f32(t, v);
    } else if (elem == QMM_ELEM_F16) {
        Vec8<F16> t;
        t.w[0] = r.a;
        vec8_to_f32(t, v);
    } else {
        Vec8<Bf16> t;
        t.w[0] = r.a;
        vec8_to_f32(t, v);
    }
}
__device__ __forceinline__ float load_elem(const void *p, int elem, int64_t i) {
    if (elem == QMM_ELEM_F32) return static_cast<const float *>(p)[i];
    if (elem == QMM_ELEM_F16) return elem_to_f32(static_cast<const F16 *>(p)[i]);
    return elem_to_f32(static_cast<const Bf16 *>(p)[i]);
}

template <typename T, int VPT, int MAXT, bool VEC>
__global__ void __launch_bounds__(MAXT) gated_norm_kernel(const qmm_gated_norm_args a, const int64_t rows_per_group) {
    __shared__ float red[4][32];
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    const int64_t row = blockIdx.x, hidden = a.hidden;
    const int64_t group = row / rows_per_group;
    const float inv_hidden = 1.0f / (float)hidden;

    auto column = [&](int i, int q) -> int64_t {
        return VEC ? (int64_t)(i * threads + tid) * 8 + q : (int64_t)(i * 8 + q) * threads + tid;
    };
    // v[i][q] = p[base + column], 0 past the row.
    auto load_row = [&](const void *p, int elem, int64_t base, float (&v)[VPT][8]) {
        if constexpr (VEC) {
            Raw8 raw[VPT];
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                raw[i] = Raw8{};
                if (column(i, 0) < hidden) raw[i] = load_raw8(p, elem, base + column(i, 0));
            }
#pragma unroll
            for (int i = 0; i < VPT; ++i) raw8_to_f32(raw[i], elem, v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int q = 0; q < 8; ++q) v[i][q] = column(i, q) < hidden ? load_elem(p, elem, base + column(i, q)) : 0.0f;
        }
    };
    int phase = 0;
    auto row_sum = [&](float s) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (warps > 1) {
            if (lane == 0) red[phase][warp] = s;
            __syncthreads();
            s = 0.0f;
            for (int w = 0; w < warps; ++w) s += red[phase][w];  // the same order in every thread
            ++phase;
        }
        return s;
    };
    // v = norm(v); columns past the row stay 0 for the sums.
    auto normalise = [&](float (&v)[VPT][8], int kind) {
        if (kind == QMM_NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int q = 0; q < 8; ++q) s += v[i][q];
            const float mean = row_sum(s) * inv_hidden;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int q = 0; q < 8; ++q) v[i][q] = column(i, q) < hidden ? v[i][q] - mean : 0.0f;
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) s = fmaf(v[i][q], v[i][q], s);
        const float r = rsqrtf(row_sum(s) * inv_hidden + a.eps);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) v[i][q] *= r;
    };

    constexpr int kElem = sizeof(T) == 4 ? (int)QMM_ELEM_F32 : 0;
    const int x_elem = sizeof(T) == 4 ? kElem : a.x_elem;
    auto store_row = [&](void *p, int64_t base, const float (&v)[VPT][8]) {
        T *o = static_cast<T *>(p) + base;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if constexpr (VEC) {
                if (column(i, 0) < hidden) store_vec8(o + column(i, 0), v[i]);
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (column(i, q) < hidden) o[column(i, q)] = elem_from_f32<T>(v[i][q]);
            }
        }
    };

    float x[VPT][8];
    load_row(a.x, x_elem, row * a.x_stride, x);
    if (a.branch) {
        float h[VPT][8], w[VPT][8], g[VPT][8];
        load_row(a.branch, a.branch_elem, row * a.branch_stride, h);
        if (a.post_weight) load_row(a.post_weight, a.vec_elem, 0, w);
        if (a.gate) load_row(a.gate, a.vec_elem, group * a.gate_stride, g);
        if (a.post != QMM_NORM_NONE) normalise(h, a.post);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float t = h[i][q];
                if (a.post_weight) t *= w[i][q];
                if (a.gate) t *= g[i][q];
                x[i][q] = fmaf(a.residual_scale, x[i][q], t);
            }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) x[i][q] *= a.residual_scale;
    }
    if (a.x_out) store_row(a.x_out, row * a.x_out_stride, x);
    if (!a.n_out && !a.n_codes) return;
    if (a.pre != QMM_NORM_NONE) normalise(x, a.pre);
    if (a.pre_weight) {
        float w[VPT][8];
        load_row(a.pre_weight, a.vec_elem, 0, w);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) x[i][q] *= w[i][q];
    }
    if (a.scale) {
        float w[VPT][8];
        load_row(a.scale, a.vec_elem, group * a.scale_stride, w);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) x[i][q] *= 1.0f + w[i][q];
    }
    if (a.shift) {
        float w[VPT][8];
        load_row(a.shift, a.vec_elem, group * a.shift_stride, w);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) x[i][q] += w[i][q];
    }
    if (a.n_out) {
        store_row(a.n_out, row * a.n_out_stride, x);
        return;
    }
    // MXFP4: columns past the row are zeros of its last block.
    const int64_t pitch = mx4_pitch(hidden), tiles = mx4_scale_tiles(hidden);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if constexpr (VEC) {
            if (column(i, 0) >= hidden) {
#pragma unroll
                for (int q = 0; q < 8; ++q) x[i][q] = 0.0f;
            }
            uint32_t codes;
            const uint32_t e = mx4_encode8(x[i], &codes);
            const int64_t c = column(i, 0);
            if (c / 2 < pitch) *reinterpret_cast<uint32_t *>(a.n_codes + row * pitch + c / 2) = codes;
            uint32_t word = e << (8 * ((lane >> 2) & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            const int64_t b = c / kMxBlock;
            if ((lane & 15) == 0 && b < tiles * 4)
                *reinterpret_cast<uint32_t *>(a.n_scales + mx4_scale_offset(row, b, tiles)) = word;
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) {  // the warp's 32 lanes hold one block
                const int64_t c = column(i, q);
                const float v = c < hidden ? x[i][q] : 0.0f;
                uint32_t m = __float_as_uint(v) & 0x7FFFFFFFu;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                const uint32_t e = mx4_scale_code(m);
                const float one[8] = {v * mx4_inverse_scale(e), 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t word = e == 255u ? 0u : (mx4_pack8(one) & 15u) << (4 * (lane & 7));
                word |= __shfl_xor_sync(0xffffffffu, word, 1);
                word |= __shfl_xor_sync(0xffffffffu, word, 2);
                word |= __shfl_xor_sync(0xffffffffu, word, 4);
                if ((lane & 7) == 0 && c / 2 < pitch) *reinterpret_cast<uint32_t *>(a.n_codes + row * pitch + c / 2) = word;
                const int64_t b = c / kMxBlock;
                if (lane == 0 && b < tiles * 4) a.n_scales[mx4_scale_offset(row, b, tiles)] = (uint8_t)e;
            }
        }
    }
}

// Threads a row: whole warps, the fewest that hold it in VPT vectors each.
template <typename T, int VPT, int MAXT, bool VEC>
static void launch_as(const qmm_gated_norm_args &a, int64_t rpg, cudaStream_t st) {
    const int64_t vectors = (a.hidden + 7) / 8;
    const unsigned threads = (unsigned)(((vectors + VPT - 1) / VPT + 31) / 32 * 32);
    gated_norm_kernel<T, VPT, MAXT, VEC><<<(unsigned)a.rows, threads, 0, st>>>(a, rpg);
}

template <typename T, bool VEC>
static void launch_vec(const qmm_gated_norm_args &a, int64_t rpg, cudaStream_t st) {
    if (a.hidden <= 1024) launch_as<T, 1, 128, VEC>(a, rpg, st);
    else if (a.hidden <= 4096) launch_as<T, 2, 256, VEC>(a, rpg, st);
    else if (a.hidden <= 8192) launch_as<T, 4, 256, VEC>(a, rpg, st);
    else if (a.hidden <= 16384) launch_as<T, 4, 512, VEC>(a, rpg, st);
    else launch_as<T, 4, 1024, VEC>(a, rpg, st);
}

}  // namespace gnorm
}  // namespace qmm

using qmm::fail;

namespace {

int64_t elem_size(int32_t e) { return e == QMM_ELEM_F32 ? 4 : 2; }
bool good_elem(int32_t e) { return e >= QMM_ELEM_BF16 && e <= QMM_ELEM_F16; }

// Bytes that `rows` rows of `cols` elements at `stride` span from p.
struct Span {
    uintptr_t lo, hi;
};
Span span_of(const void *p, int64_t rows, int64_t cols, int64_t stride, int64_t esize) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(p);
    return Span{b, b + (uintptr_t)(((rows - 1) * stride + cols) * esize)};
}
bool overlap(const Span &a, const Span &b) { return a.lo < b.hi && b.lo < a.hi; }

}  // namespace

extern "C" qmm_status qmm_gated_residual_norm(const qmm_gated_norm_args *p, void *stream) {
    if (!p) return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: null arguments");
    qmm_gated_norm_args a = *p;
    if (a.rows < 0 || a.hidden <= 0 || a.groups <= 0 || a.rows % a.groups != 0)
        return fail(QMM_ERR_BAD_SHAPE, "gated norm: %lld rows of %lld in %lld groups", (long long)a.rows, (long long)a.hidden, (long long)a.groups);
    if (a.hidden > 32768 || a.rows > INT32_MAX)
        return fail(QMM_ERR_UNSUPPORTED, "gated norm: %lld rows of %lld (at most 2^31 - 1 rows of 32768)", (long long)a.rows, (long long)a.hidden);
    if (!good_elem(a.x_elem) || !good_elem(a.branch_elem) || !good_elem(a.vec_elem))
        return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: element types %d, %d, %d", a.x_elem, a.branch_elem, a.vec_elem);
    if (a.post < QMM_NORM_NONE || a.post > QMM_NORM_LAYER || a.pre < QMM_NORM_NONE || a.pre > QMM_NORM_LAYER)
        return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: norms %d, %d", a.post, a.pre);
    if (a.rows == 0) return QMM_OK;
    if (!a.x) return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: null x");
    if (!a.branch && (a.gate || a.post_weight || a.post != QMM_NORM_NONE))
        return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: a gate or norm of the branch without a branch");
    if (!a.n_codes != !a.n_scales) return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: MXFP4 output needs codes and scales");
    if (a.n_codes && a.n_out) return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: n leaves as one form");
    const bool n = a.n_out || a.n_codes;
    if (!n && !a.x_out) return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: no output");
    if (!n && (a.pre != QMM_NORM_NONE || a.pre_weight || a.shift || a.scale))
        return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: a norm of x' without its output");
    const int64_t xs = elem_size(a.x_elem), bs = elem_size(a.branch_elem), vs = elem_size(a.vec_elem);
    if (a.rows > 1 && (a.x_stride < a.hidden || (a.branch && a.branch_stride < a.hidden) || (a.x_out && a.x_out_stride < a.hidden) ||
                       (a.n_out && a.n_out_stride < a.hidden)))
        return fail(QMM_ERR_BAD_SHAPE, "gated norm: a row stride is below %lld columns", (long long)a.hidden);
    const void *const natural[] = {a.x, a.x_out, a.n_out};
    for (const void *q : natural)
        if (reinterpret_cast<uintptr_t>(q) % xs) return fail(QMM_ERR_MISALIGNED, "gated norm: a pointer is not aligned to its element");
    const void *const vecs[] = {a.post_weight, a.pre_weight, a.gate, a.shift, a.scale};
    for (const void *q : vecs)
        if (reinterpret_cast<uintptr_t>(q) % vs) return fail(QMM_ERR_MISALIGNED, "gated norm: a vector is not aligned to its element");
    if (reinterpret_cast<uintptr_t>(a.branch) % bs) return fail(QMM_ERR_MISALIGNED, "gated norm: branch is not aligned to its element");
    if ((reinterpret_cast<uintptr_t>(a.n_codes) | reinterpret_cast<uintptr_t>(a.n_scales)) & 15)
        return fail(QMM_ERR_MISALIGNED, "gated norm: codes and scales must be 16-byte aligned");
    // An output may be an input in place: each row is read whole before it is written.
    const Span sx = span_of(a.x, a.rows, a.hidden, a.x_stride, xs);
    const Span sb = a.branch ? span_of(a.branch, a.rows, a.hidden, a.branch_stride, bs) : Span{0, 0};
    struct Out {
        const void *p;
        int64_t stride;
    } const outs[] = {{a.x_out, a.x_out_stride}, {a.n_out, a.n_out_stride}};
    for (const Out &o : outs) {
        if (!o.p) continue;
        const Span so = span_of(o.p, a.rows, a.hidden, o.stride, xs);
        if (overlap(so, sx) && !(o.p == a.x && o.stride == a.x_stride))
            return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: an output overlaps x");
        if (a.branch && overlap(so, sb) && !(o.p == a.branch && o.stride == a.branch_stride && xs == bs))
            return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: an output overlaps branch");
    }
    if (a.x_out && a.n_out && overlap(span_of(a.x_out, a.rows, a.hidden, a.x_out_stride, xs), span_of(a.n_out, a.rows, a.hidden, a.n_out_stride, xs)))
        return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: x_out overlaps n_out");
    if (a.n_codes) {
        const Span mx[] = {{reinterpret_cast<uintptr_t>(a.n_codes), reinterpret_cast<uintptr_t>(a.n_codes) + qmm_mx4_code_bytes(a.rows, a.hidden)},
                           {reinterpret_cast<uintptr_t>(a.n_scales), reinterpret_cast<uintptr_t>(a.n_scales) + qmm_mx4_scale_bytes(a.rows, a.hidden)}};
        for (const Span &m : mx)
            if (overlap(m, sx) || (a.branch && overlap(m, sb)) ||
                (a.x_out && overlap(m, span_of(a.x_out, a.rows, a.hidden, a.x_out_stride, xs))))
                return fail(QMM_ERR_INVALID_ARGUMENT, "gated norm: codes or scales overlap another operand");
    }
    const qmm_status s = qmm::check_device();
    if (s != QMM_OK) return s;

    // 16-byte accesses need every row of every operand on a 16-byte boundary.
    auto aligned = [&](const void *q, int64_t stride, int64_t esize) {
        return !q || ((reinterpret_cast<uintptr_t>(q) & 15) == 0 && (a.rows == 1 || (stride * esize) % 16 == 0));
    };
    auto aligned_vec = [&](const void *q, int64_t stride) {
        return !q || ((reinterpret_cast<uintptr_t>(q) & 15) == 0 && (a.groups == 1 || (stride * vs) % 16 == 0));
    };
    const bool vec = a.hidden % 8 == 0 && aligned(a.x, a.x_stride, xs) && aligned(a.branch, a.branch_stride, bs) &&
                     aligned(a.x_out, a.x_out_stride, xs) && aligned(a.n_out, a.n_out_stride, xs) && aligned_vec(a.post_weight, 0) &&
                     aligned_vec(a.pre_weight, 0) && aligned_vec(a.gate, a.gate_stride) && aligned_vec(a.shift, a.shift_stride) &&
                     aligned_vec(a.scale, a.scale_stride);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t rpg = a.rows / a.groups;
#define QMM_GNORM(T)                                    \
    (vec ? qmm::gnorm::launch_vec<T, true>(a, rpg, st)  \
         : qmm::gnorm::launch_vec<T, false>(a, rpg, st))
    if (a.x_elem == QMM_ELEM_F32) QMM_GNORM(float);
    else if (a.x_elem == QMM_ELEM_F16) QMM_GNORM(qmm::F16);
    else QMM_GNORM(qmm::Bf16);
#undef QMM_GNORM
    qmm::count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? QMM_OK : qmm::cuda_fail(e, "gated norm launch");
}
