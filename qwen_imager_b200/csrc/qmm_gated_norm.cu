// The seam between two sublayers of a block (qmm_gated_residual_norm):
//   h  = norm_post(branch) * post_weight
//   x' = residual_scale * x + gate * h
//   n  = norm_pre(x') * pre_weight * (1 + scale) + shift
// HBM-bound: x and branch are read once, x' and n (or its MXFP4 codes) written
// once.  A row stays in the registers of half a warp (up to 128 columns), a warp (up to
// 512) or a CTA, eight columns a vector, up to four vectors a thread, so mean and
// variance are two passes over registers, and each statistic costs one shuffle tree
// and, in a CTA, one shared slot a warp and one barrier.  The grid is what is resident
// at once, consecutive rows to a warp or CTA; it loads its next row while it works on
// this one.  Weights and modulation enter a row as three vectors, A = post_weight *
// gate, S = pre_weight * (1 + scale) and H = shift, formed once (and again where the
// group changes) in shared memory, and arithmetic goes two columns an instruction:
// with the vectors loaded and converted row by row the kernel was bound by its
// instructions (B200, 16896 x 3072 bf16: 116 us against 85; now 72, 0.88 of the measured
// HBM rate).  More rows on their way cost registers: two 101 us, three 103.
// Rows that are not 16-byte aligned are read by the aligned pieces that hold them and
// shifted into place, and stored likewise; that is bound by its instructions (4096 x
// 1677 26 us, 0.32 of HBM, x 1680 16; one element a lane at a time took 52).  Rows past
// 16384 columns, whose vectors do not fit, take a kernel without them.
#include <algorithm>
#include <type_traits>

#include "qmm_internal.h"
#include "qmm_mx4.cuh"

namespace qmm {
namespace gnorm {

// Eight elements of a 16-bit (BYTES 2) or 32-bit type, raw until used: at a 16-byte
// aligned address (VEC), or the aligned 16-byte pieces that hold them.
template <int BYTES, bool VEC>
struct Held {
    static constexpr int kBytes = BYTES, kPieces = BYTES / 2 + (VEC ? 0 : 1);
    uint4 piece[kPieces];
};
template <int BYTES>
using Raw8 = Held<BYTES, true>;
template <int BYTES>
__device__ __forceinline__ Raw8<BYTES> load_raw8(const void *p, int64_t index) {
    Raw8<BYTES> r;
    const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(p) + index * BYTES);
#pragma unroll
    for (int i = 0; i < BYTES / 2; ++i) r.piece[i] = q[i];
    return r;
}
template <int BYTES>
__device__ __forceinline__ void raw8_to_f32(const Raw8<BYTES> &r, bool f16, float (&v)[8]) {
    if constexpr (BYTES == 4) {
        Vec8<float> t;
        t.w[0] = r.piece[0];
        t.w[1] = r.piece[1];
        vec8_to_f32(t, v);
    } else if (f16) {
        Vec8<F16> t;
        t.w[0] = r.piece[0];
        vec8_to_f32(t, v);
    } else {
        Vec8<Bf16> t;
        t.w[0] = r.piece[0];
        vec8_to_f32(t, v);
    }
}
__device__ __forceinline__ float load_elem(const void *p, int elem, int64_t i) {
    if (elem == QMM_ELEM_F32) return static_cast<const float *>(p)[i];
    if (elem == QMM_ELEM_F16) return elem_to_f32(static_cast<const F16 *>(p)[i]);
    return elem_to_f32(static_cast<const Bf16 *>(p)[i]);
}

// Sums over a row, spread over the CTA's warps (SLOTS at most, a multiple of four).
// Four sets of slots taken in turn: a set is written again three barriers after its
// readers passed theirs.  The slots of warps that are not there stay 0.
template <int SLOTS, int LANES = 32>
struct RowSum {
    float (&red)[4][SLOTS];
    int set = 0;
    __device__ __forceinline__ RowSum(float (&r)[4][SLOTS]) : red(r) {
        if (LANES == 32 && blockDim.x > 32) {
            for (int i = threadIdx.x; i < 4 * SLOTS; i += blockDim.x) (&red[0][0])[i] = 0.0f;
            __syncthreads();
        }
    }
    __device__ __forceinline__ float operator()(float s) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (LANES == 32 && blockDim.x > 32) {
            if ((threadIdx.x & 31) == 0) red[set][threadIdx.x >> 5] = s;
            __syncthreads();
            s = 0.0f;
#pragma unroll
            for (int w = 0; w < SLOTS; w += 4) {  // the same order in every thread
                const float4 v = *reinterpret_cast<const float4 *>(&red[set][w]);
                s += (v.x + v.y) + (v.z + v.w);
            }
            set = (set + 1) & 3;
        }
        return s;
    }
};

// v = norm(v); columns past the row (valid(i, q) false) are 0 and stay 0.
template <int VPT, typename Sum, typename Valid>
__device__ __forceinline__ void normalise(float (&v)[VPT][8], int kind, float inv_hidden, float eps, Sum &row_sum, const Valid &valid) {
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
            for (int q = 0; q < 8; ++q) v[i][q] = valid(i, q) ? v[i][q] - mean : 0.0f;
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int q = 0; q < 8; ++q) s = fmaf(v[i][q], v[i][q], s);
    const float r = rsqrtf(row_sum(s) * inv_hidden + eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int q = 0; q < 8; ++q) v[i][q] *= r;
}

// MXFP4 of one column a lane: a warp's 32 lanes hold one block, column c this lane's.
__device__ __forceinline__ void encode_lane(const qmm_gated_norm_args &a, int64_t row, int c, float v, int64_t pitch, int64_t tiles) {
    const int lane = threadIdx.x & 31;
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

// w[0 .. N) = the words `bytes` (0 .. 15, the same in the whole warp) behind w[0].
template <int N, bool HALVES>
__device__ __forceinline__ void shift_words(uint32_t (&w)[N + 4], uint32_t bytes) {
    const bool two = bytes & 8, one = bytes & 4;
#pragma unroll
    for (int k = 0; k < N + 2; ++k) w[k] = two ? w[k + 2] : w[k];
#pragma unroll
    for (int k = 0; k < N + 1; ++k) w[k] = one ? w[k + 1] : w[k];
    if constexpr (HALVES) {
        const uint32_t s = (bytes & 2) * 8;
#pragma unroll
        for (int k = 0; k < N; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], s);
    }
}

// The row of `hidden` elements at p by the 16-byte pieces that hold it: columns [c(i),
// c(i) + 8), c(i) = first + i * step.  Its first and last piece reach into the rows
// beside it; they are not read where that would be outside [base, end), the operand.
template <int BYTES, int VPT>
__device__ __forceinline__ void fetch_pieces(Held<BYTES, false> (&held)[VPT], uintptr_t p, int first, int step, int hidden, uintptr_t base, uintptr_t end) {
    constexpr int kPieces = Held<BYTES, false>::kPieces;
    const uintptr_t a = p & ~(uintptr_t)15, past = p + (int64_t)hidden * BYTES;
    if (a >= base && ((past + 15) & ~(uintptr_t)15) <= end) {
        const int last = (int)(past - 1 - a) & ~15;  // lanes past the row read its last piece
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int k = 0; k < kPieces; ++k)
                held[i].piece[k] = *reinterpret_cast<const uint4 *>(a + min((first + i * step) * BYTES + 16 * k, last));
    } else {  // the pieces across the operand's ends: the row's elements in them, one by one
        const int lo = (int)max((int64_t)(base - p), (int64_t)-16), length = hidden * BYTES, hi = (int)min((int64_t)(end - p), (int64_t)length + 16);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const int off = (first + i * step) * BYTES + 16 * k - (int)(p - a);  // from the row's first byte
                held[i].piece[k] = make_uint4(0, 0, 0, 0);
                if (off >= lo && off + 16 <= hi) {
                    held[i].piece[k] = *reinterpret_cast<const uint4 *>(p + off);
                } else if (off < length) {
                    uint32_t w[4] = {};
#pragma unroll
                    for (int e = 0; e < 16 / BYTES; ++e) {
                        if ((uint32_t)(off + e * BYTES) < (uint32_t)length) {
                            if constexpr (BYTES == 4) w[e] = *reinterpret_cast<const uint32_t *>(p + off + e * BYTES);
                            else w[e / 2] |= (uint32_t)*reinterpret_cast<const uint16_t *>(p + off + e * BYTES) << (16 * (e & 1));
                        }
                    }
                    held[i].piece[k] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
    }
}

// Eight columns for each of LANES lanes, `count` in all, to any element-aligned address: through
// shared memory the lanes take each other's parts of the aligned 16-byte pieces, and the
// elements before the first (`skip` bytes) and after the last piece go one by one.
template <int LANES, typename T>
__device__ __forceinline__ void store_shifted(T *to, uint32_t skip, int count, const float (&v)[8], uint4 *stage) {
    constexpr int kWords = sizeof(T) * 2, kPieces = kWords / 4, kEach = 16 / sizeof(T);
    const int lane = threadIdx.x & (LANES - 1);
    uint32_t w[kWords + 4];
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
        if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
        else w[k] = pack2<T>(v[2 * k], v[2 * k + 1]);
    }
    __syncwarp();  // the stage's last readers are through
#pragma unroll
    for (int k = 0; k < kPieces; ++k) stage[lane * kPieces + k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    __syncwarp();
    const uint4 next = stage[min(lane + 1, LANES - 1) * kPieces];  // (the last lane has whole pieces only where nothing is shifted)
    w[kWords] = next.x, w[kWords + 1] = next.y, w[kWords + 2] = next.z, w[kWords + 3] = next.w;
    const int head = min((int)(skip / sizeof(T)), count), body = (count - head) / kEach;
    shift_words<kWords, sizeof(T) == 2>(w, skip);
    uint4 *const pieces = reinterpret_cast<uint4 *>(reinterpret_cast<uintptr_t>(to) + skip);
#pragma unroll
    for (int k = 0; k < kPieces; ++k)
        if (lane * kPieces + k < body) pieces[lane * kPieces + k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    const int at = lane < kEach ? lane : head + (body - 1) * kEach + lane;
    if (lane < kEach ? lane < head : lane < 2 * kEach && at < count) to[at] = reinterpret_cast<const T *>(stage)[at];
}

// blockDim.x threads a row, blockDim.y rows side by side (more than one only with 32
// threads a row).  VEC: x and branch rows, and outputs, 16-byte aligned, hidden a
// multiple of 8.
template <typename T, int BBYTES, int VPT, int MAXT, int MINB, bool VEC, int LANES>
__global__ void __launch_bounds__(MAXT, MINB)
    gated_norm_kernel(const qmm_gated_norm_args a, const uint32_t rows_per_group, const uint32_t rows_each, const bool vec_aligned) {
    extern __shared__ float4 shared_vectors[];  // A, S, H of each row side by side: threads * VPT * 8 columns (0 past the row), each thread's columns side by side
    __shared__ __align__(16) float red[4][MAXT / 32];
    __shared__ uint4 stage[VEC ? 1 : MAXT / 32][VEC ? 1 : 16 * sizeof(T)];  // a warp's own
    RowSum<MAXT / 32, LANES> row_sum{red};
    const int tid = threadIdx.x, threads = LANES == 16 ? 16 : blockDim.x, lane = tid & (LANES - 1);
    bool live = true;  // this row is one (both halves of a warp take as many turns)
    const int hidden = (int)a.hidden;
    const float inv_hidden = 1.0f / (float)hidden;
    auto column = [&](int i) { return (i * threads + tid) * 8; };
    const bool f16_branch = a.branch_elem == QMM_ELEM_F16;
    const int span = threads * VPT * 2;  // float4 a vector
    float4 *const vectors = shared_vectors + threadIdx.y * 3 * span;

    constexpr int XB = (int)sizeof(T);
    Held<XB, VEC> rx[VPT];
    Held<BBYTES, VEC> rb[VPT] = {};
    auto row_at = [](const void *p, int64_t row, int64_t stride, int bytes) { return reinterpret_cast<uintptr_t>(p) + row * stride * bytes; };
    auto fetch = [&](int64_t row) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                rx[i] = {};
                rb[i] = {};
                if (column(i) < hidden) {
                    rx[i] = load_raw8<XB>(a.x, row * a.x_stride + column(i));
                    if (a.branch) rb[i] = load_raw8<BBYTES>(a.branch, row * a.branch_stride + column(i));
                }
            }
        } else {
            auto pieces = [&](auto &held, const void *p, int64_t stride, int bytes) {
                const uintptr_t base = reinterpret_cast<uintptr_t>(p);
                fetch_pieces(held, row_at(p, row, stride, bytes), tid * 8, threads * 8, hidden, base, row_at(p, a.rows - 1, stride, bytes) + (int64_t)hidden * bytes);
            };
            pieces(rx, a.x, a.x_stride, XB);
            if (a.branch) pieces(rb, a.branch, a.branch_stride, BBYTES);
        }
    };
    // Zeroes columns past the row, which a whole vector seldom has.
    auto clear = [&](int i, float2 (&v)[4]) {
        const int left = hidden - column(i);
        if (VEC || left < 8)
        {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[q].x = (VEC ? 0 : 2 * q) >= left ? 0.0f : v[q].x;
                v[q].y = (VEC ? 0 : 2 * q + 1) >= left ? 0.0f : v[q].y;
            }
        }
    };
    auto unpack = [&](const auto &held, int i, uint32_t offset, bool f16, float2 (&v)[4]) {
        constexpr int BYTES = std::decay_t<decltype(held)>::kBytes, kPieces = std::decay_t<decltype(held)>::kPieces, kWords = BYTES * 2;
        uint32_t w[kWords + 4];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) w[4 * k] = held.piece[k].x, w[4 * k + 1] = held.piece[k].y, w[4 * k + 2] = held.piece[k].z, w[4 * k + 3] = held.piece[k].w;
        if constexpr (!VEC) shift_words<kWords, BYTES == 2>(w, offset);
        if constexpr (BYTES == 4) {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = make_float2(__uint_as_float(w[2 * q]), __uint_as_float(w[2 * q + 1]));
        } else if (f16) {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = unpack2<F16>(w[q]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = unpack2<Bf16>(w[q]);
        }
        if constexpr (!VEC) clear(i, v);
    };
    auto store = [&](void *p, int64_t base, const float2 (&v)[VPT][4]) {
        T *const o = static_cast<T *>(p) + base;
        [[maybe_unused]] const uint32_t skip = -(uint32_t)reinterpret_cast<uintptr_t>(o) & 15u;  // (a warp's columns begin at multiples of 256)
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const float w[8] = {v[i][0].x, v[i][0].y, v[i][1].x, v[i][1].y, v[i][2].x, v[i][2].y, v[i][3].x, v[i][3].y};
            const int c = column(i);
            if constexpr (VEC) {
                if (c < hidden && live) store_vec8_global(o + c, w);
            } else {
                const int from = c - lane * 8;  // the warp's first column
                if (from < hidden) store_shifted<LANES>(o + from, skip, live ? min(8 * LANES, hidden - from) : 0, w, &stage[0][0] + (threadIdx.y + tid / LANES) * (LANES * XB / 2));
            }
        }
    };
    // This thread's eight columns of vector `which`.
    auto mine = [&](int which, int i) { return vectors + which * span + i * threads * 2 + tid; };
    auto vec8 = [&](int which, int i, float2 (&w)[4]) {
        const float4 *q = mine(which, i);
        const float4 lo = q[0], hi = q[threads];
        w[0] = make_float2(lo.x, lo.y), w[1] = make_float2(lo.z, lo.w), w[2] = make_float2(hi.x, hi.y), w[3] = make_float2(hi.z, hi.w);
    };
    // Forms this thread's columns of A, S and H.
    auto take_vectors = [&](uint32_t group) {
        const int64_t gate = group * a.gate_stride, scale = group * a.scale_stride, shift = group * a.shift_stride;
#pragma unroll 1
        for (int i = 0; i < VPT; ++i) {
            auto put = [&](int k, const float (&f)[8]) {
                float4 *o = mine(k, i);
                o[0] = make_float4(f[0], f[1], f[2], f[3]);
                o[threads] = make_float4(f[4], f[5], f[6], f[7]);
            };
            if (vec_aligned) {  // every load is on its way before the first is used
                const int c = column(i);
                const bool in = VEC ? c < hidden : c + 8 <= hidden;
                auto raw = [&](const void *p, int64_t at) {
                    Raw8<4> r{};
                    if (in && p) {
                        if (a.vec_elem == QMM_ELEM_F32) r = load_raw8<4>(p, at + c);
                        else r.piece[0] = load_raw8<2>(p, at + c).piece[0];
                    }
                    return r;
                };
                auto values = [&](const Raw8<4> &r, const void *p, float none, float (&w)[8]) {
                    if (a.vec_elem == QMM_ELEM_F32) raw8_to_f32(r, false, w);
                    else raw8_to_f32(Raw8<2>{{r.piece[0]}}, a.vec_elem == QMM_ELEM_F16, w);
                    if (!p) {
#pragma unroll
                        for (int q = 0; q < 8; ++q) w[q] = none;
                    }
                };
                const Raw8<4> r0 = raw(a.post_weight, 0), r1 = raw(a.gate, gate), r2 = raw(a.pre_weight, 0), r3 = raw(a.scale, scale), r4 = raw(a.shift, shift);
                const float one = in ? 1.0f : 0.0f;
                float f[8], w[8];
                values(r0, a.post_weight, one, f);
                values(r1, a.gate, 1.0f, w);
#pragma unroll
                for (int q = 0; q < 8; ++q) f[q] *= w[q];
                put(0, f);
                values(r2, a.pre_weight, one, f);
                values(r3, a.scale, 0.0f, w);
#pragma unroll
                for (int q = 0; q < 8; ++q) f[q] = fmaf(f[q], w[q], f[q]);
                put(1, f);
                values(r4, a.shift, 0.0f, f);
                put(2, f);
                const int col = (hidden & ~7) + lane;
                if (!VEC && c - lane * 8 < hidden && (hidden & 7) != 0 && c - lane * 8 + 8 * LANES >= hidden) {  // the row's last vector: a column a lane
                    const uint32_t lanes = LANES == 16 ? 0xFFFFu << (threadIdx.y & 1) * 16 : 0xFFFFFFFFu;
                    __syncwarp(lanes);
                    if (col < hidden) {
                        auto at = [&](const void *p, int64_t base, float none) { return p ? load_elem(p, a.vec_elem, base + col) : none; };
                        const float v = at(a.pre_weight, 0, 1.0f);
                        float *const o = reinterpret_cast<float *>(vectors + i * threads + (col & 4 ? threads : 0) + (col >> 3)) + (col & 3);
                        o[0] = at(a.post_weight, 0, 1.0f) * at(a.gate, gate, 1.0f);
                        o[span * 4] = fmaf(v, at(a.scale, scale, 0.0f), v);
                        o[span * 8] = at(a.shift, shift, 0.0f);
                    }
                    __syncwarp(lanes);
                }
            } else {
                // One element at a time, the loads of four columns on their way together.
                auto value = [&](uint32_t w) {
                    return a.vec_elem == QMM_ELEM_F32 ? __uint_as_float(w) : a.vec_elem == QMM_ELEM_F16 ? elem_to_f32(F16{(uint16_t)w}) : elem_to_f32(Bf16{(uint16_t)w});
                };
#pragma unroll(VEC ? 1 : 2)
                for (int half = 0; half < 2; ++half) {
                    const int c = column(i) + 4 * half;
                    auto raw = [&](const void *p, int64_t at, uint32_t (&w)[4]) {
                        const int n = p ? hidden - c : 0;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            w[q] = 0;
                            if (q < n) w[q] = a.vec_elem == QMM_ELEM_F32 ? static_cast<const uint32_t *>(p)[at + c + q] : static_cast<const uint16_t *>(p)[at + c + q];
                        }
                    };
                    uint32_t r[5][4];
                    raw(a.post_weight, 0, r[0]), raw(a.gate, gate, r[1]), raw(a.pre_weight, 0, r[2]), raw(a.scale, scale, r[3]), raw(a.shift, shift, r[4]);
                    float f[3][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float one = c + q < hidden ? 1.0f : 0.0f, w = a.pre_weight ? value(r[2][q]) : one;
                        f[0][q] = (a.post_weight ? value(r[0][q]) : one) * (a.gate ? value(r[1][q]) : 1.0f);
                        f[1][q] = fmaf(w, value(r[3][q]), w);
                        f[2][q] = value(r[4][q]);
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k) mine(k, i)[half * threads] = make_float4(f[k][0], f[k][1], f[k][2], f[k][3]);
                }
            }
        }
    };
    // v -= mean, for the sums of squares of a layer norm (columns past the row stay 0).
    auto centre = [&](float2 (&v)[VPT][4]) {
        float2 s = twice(0.0f);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) s = add_f32x2(s, v[i][q]);
        const float mean = row_sum(s.x + s.y) * inv_hidden;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) v[i][q] = add_f32x2(v[i][q], twice(VEC && column(i) >= hidden ? 0.0f : -mean));
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) clear(i, v[i]);
        }
    };
    auto rms = [&](const float2 (&v)[VPT][4]) {
        float2 s = twice(0.0f);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) s = fma_f32x2(v[i][q], v[i][q], s);
        return rsqrtf(row_sum(s.x + s.y) * inv_hidden + a.eps);
    };
    const int64_t pitch = mx4_pitch(hidden), tiles = mx4_scale_tiles(hidden);

    pdl_launch_dependents();  // a product behind this pass sets itself up meanwhile; it waits for the grid before it reads
    const uint32_t first = (blockIdx.x * blockDim.y + threadIdx.y) * rows_each, last = min(first + rows_each, (uint32_t)a.rows);
    if (first < last) fetch(first);
    uint32_t group_end = first;
    const uint32_t end = LANES == 16 ? first + rows_each : last;
    for (uint32_t row = first; row < end; ++row) {
        if constexpr (LANES == 16) live = row < last;
        if (live && row == group_end) {
            const uint32_t group = row / rows_per_group;
            group_end = (group + 1) * rows_per_group;
            take_vectors(group);
        }
        float2 x[VPT][4], h[VPT][4];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            unpack(rx[i], i, VEC ? 0u : (uint32_t)row_at(a.x, row, a.x_stride, XB) & 15u, std::is_same<T, F16>::value, x[i]);
            unpack(rb[i], i, VEC ? 0u : (uint32_t)row_at(a.branch, row, a.branch_stride, BBYTES) & 15u, f16_branch, h[i]);
        }
        if (row + 1 < last) fetch((int64_t)row + 1);
        const float2 c2 = twice(a.residual_scale);
        if (a.branch) {
            if (a.post == QMM_NORM_LAYER) centre(h);
            const float2 r = twice(a.post != QMM_NORM_NONE ? rms(h) : 1.0f);
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                float2 w[4];
                vec8(0, i, w);
#pragma unroll
                for (int q = 0; q < 4; ++q) x[i][q] = fma_f32x2(x[i][q], c2, mul_f32x2(mul_f32x2(h[i][q], r), w[q]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) x[i][q] = mul_f32x2(x[i][q], c2);
        }
        if (a.x_out) store(a.x_out, row * a.x_out_stride, x);
        if (!a.n_out && !a.n_codes) continue;
        if (a.pre == QMM_NORM_LAYER) centre(x);
        const float2 r = twice(a.pre != QMM_NORM_NONE ? rms(x) : 1.0f);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            float2 w[4], s[4];
            vec8(1, i, w);
            vec8(2, i, s);
#pragma unroll
            for (int q = 0; q < 4; ++q) x[i][q] = fma_f32x2(mul_f32x2(x[i][q], r), w[q], s[q]);
        }
        if (a.n_out) {
            store(a.n_out, row * a.n_out_stride, x);
            continue;
        }
        // MXFP4: columns past the row are zeros of its last block.
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            clear(i, x[i]);  // (0 times an infinite or NaN statistic)
            float w[8] = {x[i][0].x, x[i][0].y, x[i][1].x, x[i][1].y, x[i][2].x, x[i][2].y, x[i][3].x, x[i][3].y};
            const int c = column(i);
            uint32_t codes;
            const uint32_t e = mx4_encode8(w, &codes);
            if (c / 2 < pitch && live) *reinterpret_cast<uint32_t *>(a.n_codes + row * pitch + c / 2) = codes;
            uint32_t word = e << (8 * ((lane >> 2) & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            const int64_t b = c / kMxBlock;
            if ((lane & 15) == 0 && b < tiles * 4 && live) {
                *reinterpret_cast<uint32_t *>(a.n_scales + mx4_scale_offset(row, b, tiles)) = word;
                if (LANES == 16) *reinterpret_cast<uint32_t *>(a.n_scales + mx4_scale_offset(row, 4, tiles)) = 0;
            }
        }
    }
}

// Any alignment and width, nothing kept between rows.  A row of up to 32768 columns in 1024
// threads leaves 64 registers a thread, so that x and h spill (B200, 1024 x 20000 bf16 249 us,
// 0.10 of the measured HBM rate; f32 193, 0.26).
template <typename T, int VPT, int MAXT>
__global__ void __launch_bounds__(MAXT) gated_norm_any_kernel(const qmm_gated_norm_args a, const uint32_t rows_per_group) {
    __shared__ __align__(16) float red[4][MAXT / 32];
    RowSum<MAXT / 32> row_sum{red};
    const int tid = threadIdx.x, threads = blockDim.x;
    const int64_t row = blockIdx.x;
    const int hidden = (int)a.hidden;
    const int64_t group = (uint32_t)row / rows_per_group;
    const float inv_hidden = 1.0f / (float)hidden;
    auto column = [&](int i, int q) { return (i * 8 + q) * threads + tid; };
    auto valid = [&](int i, int q) { return column(i, q) < hidden; };
    auto load = [&](const void *p, int elem, int64_t base, float (&v)[VPT][8]) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) v[i][q] = valid(i, q) ? load_elem(p, elem, base + column(i, q)) : 0.0f;
    };
    auto store = [&](void *p, int64_t base, const float (&v)[VPT][8]) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (valid(i, q)) static_cast<T *>(p)[base + column(i, q)] = elem_from_f32<T>(v[i][q]);
    };
    auto with = [&](const void *vec, int64_t base, float (&v)[VPT][8], auto f) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (valid(i, q)) v[i][q] = f(v[i][q], load_elem(vec, a.vec_elem, base + column(i, q)));
    };
    float x[VPT][8], h[VPT][8];
    load(a.x, a.x_elem, row * a.x_stride, x);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int q = 0; q < 8; ++q) h[i][q] = 0.0f;
    if (a.branch) {
        load(a.branch, a.branch_elem, row * a.branch_stride, h);
        if (a.post != QMM_NORM_NONE) normalise(h, a.post, inv_hidden, a.eps, row_sum, valid);
        if (a.post_weight) with(a.post_weight, 0, h, [](float v, float w) { return v * w; });
        if (a.gate) with(a.gate, group * a.gate_stride, h, [](float v, float w) { return v * w; });
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int q = 0; q < 8; ++q) x[i][q] = fmaf(a.residual_scale, x[i][q], h[i][q]);
    if (a.x_out) store(a.x_out, row * a.x_out_stride, x);
    if (!a.n_out && !a.n_codes) return;
    if (a.pre != QMM_NORM_NONE) normalise(x, a.pre, inv_hidden, a.eps, row_sum, valid);
    if (a.pre_weight) with(a.pre_weight, 0, x, [](float v, float w) { return v * w; });
    if (a.scale) with(a.scale, group * a.scale_stride, x, [](float v, float w) { return fmaf(v, w, v); });
    if (a.shift) with(a.shift, group * a.shift_stride, x, [](float v, float w) { return v + w; });
    if (a.n_out) {
        store(a.n_out, row * a.n_out_stride, x);
        return;
    }
    // MXFP4: columns past the row are zeros of its last block.
    const int64_t pitch = mx4_pitch(hidden), tiles = mx4_scale_tiles(hidden);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int q = 0; q < 8; ++q) encode_lane(a, row, column(i, q), valid(i, q) ? x[i][q] : 0.0f, pitch, tiles);
}

// Threads a row: whole warps, the fewest that hold it in VPT vectors each.
template <int VPT>
static unsigned threads_for(int64_t hidden) {
    const int64_t vectors = (hidden + 7) / 8;
    return (unsigned)(((vectors + VPT - 1) / VPT + 31) / 32 * 32);
}

template <typename T, int BBYTES, int VPT, int MAXT, int MINB, bool VEC, int LANES = 32>
static cudaError_t launch_rows(const qmm_gated_norm_args &a, uint32_t rpg, bool vec_aligned, cudaStream_t st) {
    auto kernel = gated_norm_kernel<T, BBYTES, VPT, MAXT, MINB, VEC, LANES>;
    const unsigned threads = LANES == 16 ? 16 : threads_for<VPT>(a.hidden);
    const dim3 block(threads, threads <= 32 ? 128 / threads : 1, 1);
    const size_t smem = (size_t)threads * block.y * VPT * 8 * 4 * 3;
    static int resident[64][33] = {};  // CTAs an SM by device and warps a row
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    int &n = resident[dev][threads / 32];
    if (n == 0) {
        int m = 0;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAXT * VPT * 8 * 4 * 3);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&m, kernel, (int)(threads * block.y), smem);
        if (e != cudaSuccess) return e;
        n = std::max(1, m);
    }
    // Consecutive rows to a warp or CTA: few of them cross into another group's vectors.
    const int64_t places = (int64_t)sm_count() * n * block.y, each = (a.rows + places - 1) / places;
    const int64_t used = (a.rows + each - 1) / each;
    kernel<<<(unsigned)((used + block.y - 1) / block.y), block, smem, st>>>(a, rpg, (uint32_t)each, vec_aligned);
    return cudaGetLastError();
}

template <typename T, int BBYTES, bool VEC>
static cudaError_t launch_fast(const qmm_gated_norm_args &a, uint32_t rpg, bool vec_aligned, cudaStream_t st) {
    // Half a warp or a warp a row where its lanes hold it (B200, 30000 x 128 bf16: half a
    // warp 8.7 us, a warp 14.6); then a CTA, with as many vectors a thread as its registers
    // allow at 12 warps an SM or more (16896 x 2048: two vectors a thread 70 us, one 77).
    constexpr bool W = sizeof(T) == 4 || BBYTES == 4 || !VEC;  // more registers a vector
    if (a.hidden <= 128) return launch_rows<T, BBYTES, 1, 256, W ? 3 : 4, VEC, 16>(a, rpg, vec_aligned, st);
    if (a.hidden <= 256) return launch_rows<T, BBYTES, 1, 256, W ? 3 : 4, VEC>(a, rpg, vec_aligned, st);
    if (a.hidden <= 4096) return launch_rows<T, BBYTES, 2, 256, W ? 2 : 3, VEC>(a, rpg, vec_aligned, st);
    if (VEC && a.hidden <= 8192) return launch_rows<T, BBYTES, 4, 256, W ? 1 : 2, true>(a, rpg, vec_aligned, st);
    if (!VEC && a.hidden <= 8192) return launch_rows<T, BBYTES, 2, 512, 1, false>(a, rpg, vec_aligned, st);
    return launch_rows<T, BBYTES, 4, 512, 1, VEC>(a, rpg, vec_aligned, st);
}

template <typename T>
static cudaError_t launch(const qmm_gated_norm_args &a, bool vec, bool vec_aligned, uint32_t rpg, cudaStream_t st) {
    if (a.hidden > 16384) {
        gated_norm_any_kernel<T, 4, 1024><<<(unsigned)a.rows, threads_for<4>(a.hidden), 0, st>>>(a, rpg);
        return cudaGetLastError();
    }
    const bool wide_branch = a.branch_elem == QMM_ELEM_F32;
    if (vec) return wide_branch ? launch_fast<T, 4, true>(a, rpg, vec_aligned, st) : launch_fast<T, 2, true>(a, rpg, vec_aligned, st);
    return wide_branch ? launch_fast<T, 4, false>(a, rpg, vec_aligned, st) : launch_fast<T, 2, false>(a, rpg, vec_aligned, st);
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
    const bool vec_aligned = aligned_vec(a.post_weight, 0) && aligned_vec(a.pre_weight, 0) && aligned_vec(a.gate, a.gate_stride) &&
                             aligned_vec(a.shift, a.shift_stride) && aligned_vec(a.scale, a.scale_stride);
    const bool vec = a.hidden % 8 == 0 && aligned(a.x, a.x_stride, xs) && aligned(a.branch, a.branch_stride, bs) &&
                     aligned(a.x_out, a.x_out_stride, xs) && aligned(a.n_out, a.n_out_stride, xs);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint32_t rpg = (uint32_t)(a.rows / a.groups);
    const cudaError_t e = a.x_elem == QMM_ELEM_F32   ? qmm::gnorm::launch<float>(a, vec, vec_aligned, rpg, st)
                          : a.x_elem == QMM_ELEM_F16 ? qmm::gnorm::launch<qmm::F16>(a, vec, vec_aligned, rpg, st)
                                                     : qmm::gnorm::launch<qmm::Bf16>(a, vec, vec_aligned, rpg, st);
    qmm::count_launch();
    return e == cudaSuccess ? QMM_OK : qmm::cuda_fail(e, "gated norm launch");
}
