// RMSNorm per head of q and k, and rotary positions with several axes
// (qmm_qk_norm_rotary).
//
// HBM-bound: q and k are read and written once; positions are a few bytes a
// token.  A warp takes a token and a run of its heads.  Each lane holds the same
// four pairs of every head (as two runs of four columns), so the token's sines
// and cosines, computed once in the warp (a pair or two a lane, handed round by
// shuffles) and multiplied with the norm's weight, stay in registers over the
// heads; a head of 8 U columns takes U lanes, and 32 / U heads (rounded down) go at a
// time.  Arithmetic goes two columns an instruction.
//
// The angle is positions * turns in turns.  With turns = f + g (leading and
// trailing term), p = fl(pos f) and e = pos f - p exact by one fma, the fraction
// of p is exact and the angle's error stays near 2^-24 turns up to positions of 2^24.
// Past these a whole position is two terms too, each product gives up its whole
// turns, and what g lacks of the frequency decides: 2^-52 of the position, for
// frequencies up to a radian (2^-21 turns at 2^31).
#include "qmm_internal.h"
#include "qmm_mx4.cuh"

namespace qmm {
namespace rotary {

constexpr int kWarps = 4;
// CTAs an SM: 32 warps cover the loads (B200, 16896 x 48 heads x 128 bf16: 72 us, 0.88 of
// the measured HBM rate, 70 where operands stay the same; before lanes shared their sines 73, with 16 warps 95, with 40 79).
constexpr int kResident = 8;

// A position as two terms: whole numbers past 2^24 do not fit one.
__device__ __forceinline__ float position_of(const qmm_rotary_args &a, int64_t batch, int64_t token, int axis, float *low) {
    const int64_t i = batch * a.pos_batch_stride + token * a.axes + axis;
    *low = 0.0f;
    if (a.pos_kind == 2) return static_cast<const float *>(a.positions)[i];
    const int64_t v = a.pos_kind == 0 ? static_cast<const int32_t *>(a.positions)[i] : static_cast<const int64_t *>(a.positions)[i];
    const float high = (float)v;
    *low = (float)(v - (int64_t)high);
    return high;
}

__device__ __forceinline__ float fraction(float x) { return x - rintf(x); }

__device__ __forceinline__ void pair_turn(const qmm_rotary_args &a, int64_t batch, int64_t token, int pair, float *c, float *s) {
    float low;
    const float pos = position_of(a, batch, token, a.axis[pair], &low);
    const float f = a.turns[2 * pair], g = a.turns[2 * pair + 1];
    const float p = pos * f;
    const float e = fmaf(pos, f, -p);
    float t;
    if (fabsf(pos) <= 16777216.0f && low == 0.0f) {
        t = fraction(p) + fmaf(pos, g, e);
    } else {
        const float pg = pos * g, pl = low * f;
        const float small = fmaf(pos, g, -pg) + fmaf(low, f, -pl) + low * g;
        t = fraction(p) + fraction(e) + fraction(pg) + fraction(pl) + small;
    }
    sincospif(2.0f * t, s, c);
}

// How a lane's eight columns lie: one run of eight with adjacent pairs, at an address
// aligned to eight elements; the same aligned to four; two runs of four (halves).
enum Layout { kWide, kAdjacent, kHalves };

template <typename T>
struct Runs {
    uint32_t w[sizeof(T) * 2];
};
template <typename T, Layout L>
__device__ __forceinline__ Runs<T> load_runs(const T *p, int ca, int cb) {
    Runs<T> r;
    if constexpr (sizeof(T) == 4) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p + ca), b = *reinterpret_cast<const uint4 *>(p + cb);
        r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
        r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
    } else if constexpr (L == kWide) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p + ca);
        r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
    } else {
        const uint2 a = *reinterpret_cast<const uint2 *>(p + ca), b = *reinterpret_cast<const uint2 *>(p + cb);
        r.w[0] = a.x, r.w[1] = a.y, r.w[2] = b.x, r.w[3] = b.y;
    }
    return r;
}
// The first and second members of the lane's four pairs, two pairs a float2.
template <typename T, Layout L>
__device__ __forceinline__ void runs_to_pairs(const Runs<T> &r, float2 (&a)[2], float2 (&b)[2]) {
    float v[8];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(r.w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (L == kHalves) {
            a[i] = make_float2(v[2 * i], v[2 * i + 1]);
            b[i] = make_float2(v[4 + 2 * i], v[4 + 2 * i + 1]);
        } else {
            a[i] = make_float2(v[4 * i], v[4 * i + 2]);
            b[i] = make_float2(v[4 * i + 1], v[4 * i + 3]);
        }
    }
}
// The inverse, word for word.
template <typename T, Layout L>
__device__ __forceinline__ Runs<T> pairs_to_runs(const float2 (&a)[2], const float2 (&b)[2]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (L == kHalves) {
            v[2 * i] = a[i].x, v[2 * i + 1] = a[i].y;
            v[4 + 2 * i] = b[i].x, v[4 + 2 * i + 1] = b[i].y;
        } else {
            v[4 * i] = a[i].x, v[4 * i + 2] = a[i].y;
            v[4 * i + 1] = b[i].x, v[4 * i + 3] = b[i].y;
        }
    }
    Runs<T> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
    return r;
}
template <typename T, Layout L>
__device__ __forceinline__ void store_runs(T *p, int ca, int cb, const Runs<T> &r) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint4 *>(p + ca) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
        *reinterpret_cast<uint4 *>(p + cb) = make_uint4(r.w[4], r.w[5], r.w[6], r.w[7]);
    } else if constexpr (L == kWide) {
        *reinterpret_cast<uint4 *>(p + ca) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    } else {
        *reinterpret_cast<uint2 *>(p + ca) = make_uint2(r.w[0], r.w[1]);
        *reinterpret_cast<uint2 *>(p + cb) = make_uint2(r.w[2], r.w[3]);
    }
}

// The heads [h0, h1) of one operand for one token.
template <typename T>
struct Heads {
    const T *src;
    T *dst;
    int64_t src_stride, dst_stride;
    int h0, h1;
};

// A warp takes a token and a run of its q and k heads.  Needs dim % 8 == 0, with
// halves pairs % 4 == 0, heads aligned as the layout says.  NORM: some weight is
// given; POW2: dim / 8 is a power of two; TAIL: some columns are not turned.  A turn by 0
// would mix an infinity or NaN of one into its lane's neighbour (0 times either is NaN),
// so without a norm their words leave as they came, and with one selects keep them apart
// (B200, 2 x 14317 x 24 x 72 f16 41.0 -> 42.5 us; with a norm, 16896 x 48 x 128 with 32 of
// 64 pairs 71.6 -> 75.8, in halves 77.8 -> 80.7; a branch on the head's sum of squares and
// predicated products cost registers and as much time).
template <typename T, Layout L, bool NORM, bool POW2, bool TAIL, int kTurns>
__global__ void __launch_bounds__(kWarps * 32, kResident) rotary_kernel(const qmm_rotary_args a, const int heads_per_warp) {
    constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;  // heads a lane group has in flight
    const int units = a.dim >> 3, at_a_time = 32 / units;
    const int lane = threadIdx.x & 31, sub = lane / units, u = lane - sub * units;
    const uint32_t row = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= (uint32_t)(a.batch * a.tokens)) return;
    const uint32_t tokens = (uint32_t)a.tokens, batch = row / tokens, token = row - batch * tokens;
    const int first = blockIdx.y * heads_per_warp, last = first + heads_per_warp;
    const bool live = sub < at_a_time;
    const int pair = u * 4;
    const int ca = L == kHalves && pair < a.pairs ? pair : u * 8, cb = L == kHalves && pair < a.pairs ? a.pairs + pair : u * 8 + 4;
    const float inv_dim = 1.0f / (float)a.dim;
    auto turns = [&](int i) { return pair + (L == kHalves ? 0 : i) < a.pairs; };  // pair i of the lane (halves: all four or none)
    float2 cs[2], sn[2];
    bool turned = false;

    auto run = [&](const Heads<T> &h, const void *weight) {
        if (h.h0 >= h.h1) return;
        const T *src = h.src + (int64_t)(h.h0 + sub) * h.src_stride;
        T *dst = h.dst + (int64_t)(h.h0 + sub) * h.dst_stride;
        const int64_t src_step = at_a_time * h.src_stride, dst_step = at_a_time * h.dst_stride;
        int left = live ? h.h1 - h.h0 - sub : 0;  // heads from this lane's on
        // first = r (x A + y B), second = r (x C + y D): the norm's weights and the turn in one factor
        float2 fa[2], fb[2], fc[2], fd[2];
        for (int hb = h.h0; hb < h.h1; hb += at_a_time * kAhead) {
            Runs<T> raw[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                raw[j] = Runs<T>{};
                if (j * at_a_time < left) raw[j] = load_runs<T, L>(src + j * src_step, ca, cb);
            }
            if (!turned) {  // (while the first heads are on their way)
                turned = true;
                // Each lane turns pairs lane, lane + 32, ... and takes its four from the lanes that have them.
                float c[kTurns], v[kTurns];
#pragma unroll
                for (int j = 0; j < kTurns; ++j) {
                    c[j] = 1.0f, v[j] = 0.0f;
                    if (lane + 32 * j < a.pairs) pair_turn(a, batch, token, lane + 32 * j, &c[j], &v[j]);
                }
                float mc[4], ms[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    mc[i] = 1.0f, ms[i] = 0.0f;
#pragma unroll
                    for (int j = 0; j < kTurns; ++j) {
                        const float tc = __shfl_sync(0xffffffffu, c[j], (pair + i) & 31), ts = __shfl_sync(0xffffffffu, v[j], (pair + i) & 31);
                        if ((pair + i) >> 5 == j) mc[i] = tc, ms[i] = ts;
                    }
                }
                cs[0] = make_float2(mc[0], mc[1]), cs[1] = make_float2(mc[2], mc[3]);
                sn[0] = make_float2(ms[0], ms[1]), sn[1] = make_float2(ms[2], ms[3]);
            }
            if (hb == h.h0) {
                float2 we[2] = {twice(1.0f), twice(1.0f)}, wo[2] = {twice(1.0f), twice(1.0f)};
                if (NORM && weight && live) runs_to_pairs<T, L>(load_runs<T, L>(static_cast<const T *>(weight), ca, cb), we, wo);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    fa[i] = mul_f32x2(we[i], cs[i]);
                    fb[i] = mul_f32x2(wo[i], make_float2(-sn[i].x, -sn[i].y));
                    fc[i] = mul_f32x2(we[i], sn[i]);
                    fd[i] = mul_f32x2(wo[i], cs[i]);
                    if (TAIL && NORM && !turns(2 * i)) fb[i].x = fc[i].x = -0.0f;  // 0 * -0 changes no number that it is added to
                    if (TAIL && NORM && !turns(2 * i + 1)) fb[i].y = fc[i].y = -0.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (hb + j * at_a_time >= h.h1) break;
                float2 x[2], y[2];
                runs_to_pairs<T, L>(raw[j], x, y);
                if (NORM && weight) {
                    float2 p = mul_f32x2(x[0], x[0]);
                    p = fma_f32x2(x[1], x[1], p);
                    p = fma_f32x2(y[0], y[0], p);
                    p = fma_f32x2(y[1], y[1], p);
                    float s = p.x + p.y;
                    if constexpr (POW2) {
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1)
                            if (o < units) s += __shfl_xor_sync(0xffffffffu, s, o);
                    } else {  // lanes u .. of the head's units, then the first one's sum
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            if (o < units) {
                                const float t = __shfl_down_sync(0xffffffffu, s, o);
                                if (u + o < units) s += t;
                            }
                        }
                        s = __shfl_sync(0xffffffffu, s, lane - u);
                    }
                    const float2 r = twice(rsqrtf(s * inv_dim + a.eps));
#pragma unroll
                    for (int q = 0; q < 2; ++q) x[q] = mul_f32x2(x[q], r), y[q] = mul_f32x2(y[q], r);
                }
                if (j * at_a_time < left) {
                    float2 oa[2], ob[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float2 xc = x[q], yc = y[q];
                        if constexpr (TAIL && NORM) {
                            const bool first = turns(2 * q), second = turns(2 * q + 1);
                            xc = make_float2(first ? xc.x : 0.0f, second ? xc.y : 0.0f);
                            yc = make_float2(first ? yc.x : 0.0f, second ? yc.y : 0.0f);
                        }
                        oa[q] = fma_f32x2(x[q], fa[q], mul_f32x2(yc, fb[q]));
                        ob[q] = fma_f32x2(xc, fc[q], mul_f32x2(y[q], fd[q]));
                    }
                    Runs<T> out = pairs_to_runs<T, L>(oa, ob);
                    if constexpr (TAIL && !NORM) {
#pragma unroll
                        for (int i = 0; i < (int)sizeof(T) * 2; ++i) out.w[i] = turns(i * 2 / (int)sizeof(T)) ? out.w[i] : raw[j].w[i];
                    }
                    store_runs<T, L>(dst + j * dst_step, ca, cb, out);
                }
            }
            src += src_step * kAhead;
            dst += dst_step * kAhead;
            left -= at_a_time * kAhead;
        }
    };
    run(Heads<T>{static_cast<const T *>(a.q) + batch * a.q_stride[0] + token * a.q_stride[1],
                 static_cast<T *>(a.q_out) + batch * a.q_out_stride[0] + token * a.q_out_stride[1], a.q_stride[2], a.q_out_stride[2],
                 first, min(last, a.q_heads)},
        a.q_weight);
    run(Heads<T>{static_cast<const T *>(a.k) + batch * a.k_stride[0] + token * a.k_stride[1],
                 static_cast<T *>(a.k_out) + batch * a.k_out_stride[0] + token * a.k_out_stride[1], a.k_stride[2], a.k_out_stride[2],
                 max(first - a.q_heads, 0), min(last - a.q_heads, a.k_heads)},
        a.k_weight);
}

// Any dim up to 256, any pairs, any alignment: lane l takes pairs l, l + 32, ...
// and the unrotated columns likewise, element by element, one head at a time.  Bound by
// its narrow accesses (B200, 16896 x 48 x 128 bf16 in halves with 31 pairs 315 us, 0.20 of
// the measured HBM rate).
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) rotary_any_kernel(const qmm_rotary_args a, const int heads_per_warp) {
    const int lane = threadIdx.x & 31;
    const uint32_t row = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= (uint32_t)(a.batch * a.tokens)) return;
    const uint32_t tokens = (uint32_t)a.tokens, batch = row / tokens, token = row - batch * tokens;
    const int heads = a.q_heads + a.k_heads;
    const int h0 = blockIdx.y * heads_per_warp, h1 = min(h0 + heads_per_warp, heads);
    float cs[4], sn[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        cs[j] = 1.0f, sn[j] = 0.0f;
        if (lane + 32 * j < a.pairs) pair_turn(a, batch, token, lane + 32 * j, &cs[j], &sn[j]);
    }
    const float inv_dim = 1.0f / (float)a.dim;
    for (int h = h0; h < h1; ++h) {
        const bool isq = h < a.q_heads;
        const int hh = isq ? h : h - a.q_heads;
        const T *src = isq ? static_cast<const T *>(a.q) + batch * a.q_stride[0] + token * a.q_stride[1] + hh * a.q_stride[2]
                           : static_cast<const T *>(a.k) + batch * a.k_stride[0] + token * a.k_stride[1] + hh * a.k_stride[2];
        T *dst = isq ? static_cast<T *>(a.q_out) + batch * a.q_out_stride[0] + token * a.q_out_stride[1] + hh * a.q_out_stride[2]
                     : static_cast<T *>(a.k_out) + batch * a.k_out_stride[0] + token * a.k_out_stride[1] + hh * a.k_out_stride[2];
        const T *w = static_cast<const T *>(isq ? a.q_weight : a.k_weight);
        float va[4], vb[4], rest[8];
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = lane + 32 * j;
            va[j] = vb[j] = 0.0f;
            if (p < a.pairs) {
                va[j] = elem_to_f32(src[a.adjacent ? 2 * p : p]);
                vb[j] = elem_to_f32(src[a.adjacent ? 2 * p + 1 : a.pairs + p]);
            }
            s = fmaf(va[j], va[j], fmaf(vb[j], vb[j], s));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = 2 * a.pairs + lane + 32 * j;
            rest[j] = c < a.dim ? elem_to_f32(src[c]) : 0.0f;
            s = fmaf(rest[j], rest[j], s);
        }
        float r = 1.0f;
        if (w) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            r = rsqrtf(s * inv_dim + a.eps);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int p = lane + 32 * j;
            if (p < a.pairs) {
                const int ia = a.adjacent ? 2 * p : p, ib = a.adjacent ? 2 * p + 1 : a.pairs + p;
                const float x = w ? va[j] * (r * elem_to_f32(w[ia])) : va[j], y = w ? vb[j] * (r * elem_to_f32(w[ib])) : vb[j];
                dst[ia] = elem_from_f32<T>(x * cs[j] - y * sn[j]);
                dst[ib] = elem_from_f32<T>(x * sn[j] + y * cs[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = 2 * a.pairs + lane + 32 * j;
            if (c < a.dim) dst[c] = elem_from_f32<T>(w ? rest[j] * (r * elem_to_f32(w[c])) : rest[j]);
        }
        __syncwarp();
    }
}

template <typename T>
static qmm_status launch(const qmm_rotary_args &a, bool fast, bool wide, cudaStream_t st) {
    const int heads = a.q_heads + a.k_heads, units = a.dim / 8;
    const int at_a_time = fast ? 32 / units : 1;
    // Heads a warp: all of a token's where the tokens alone fill the machine, so
    // that its sines are computed once; fewer where they do not, down to the
    // heads that a warp handles at a time.
    const int64_t rows = a.batch * a.tokens;
    if (rows > INT32_MAX) return fail(QMM_ERR_UNSUPPORTED, "rotary: %lld tokens are past the launch limits", (long long)rows);
    const int64_t most = (heads + at_a_time - 1) / at_a_time;
    int64_t splits = 1;
    while (splits < most && rows * splits < (int64_t)sm_count() * 16) splits *= 2;
    if (splits > most) splits = most;
    int per = (int)((heads + splits - 1) / splits);
    per = (per + at_a_time - 1) / at_a_time * at_a_time;
    const dim3 grid((unsigned)((rows + kWarps - 1) / kWarps), (unsigned)((heads + per - 1) / per), 1);
    if (grid.y > 65535) return fail(QMM_ERR_UNSUPPORTED, "rotary: %d heads are past the launch limits", heads);
    const bool norm = a.q_weight || a.k_weight, pow2 = (units & (units - 1)) == 0;
#define QMM_ROTARY(L)                                                                            \
    (a.pairs <= 32 ? QMM_ROTARY_N(L, 1) : a.pairs <= 64 ? QMM_ROTARY_N(L, 2) : QMM_ROTARY_N(L, 4))
#define QMM_ROTARY_N(L, N) (2 * a.pairs < a.dim ? QMM_ROTARY_T(L, true, N) : QMM_ROTARY_T(L, false, N))
#define QMM_ROTARY_T(L, TAIL, N)                                                                 \
    (!norm  ? rotary_kernel<T, L, false, true, TAIL, N><<<grid, kWarps * 32, 0, st>>>(a, per)    \
     : pow2 ? rotary_kernel<T, L, true, true, TAIL, N><<<grid, kWarps * 32, 0, st>>>(a, per)     \
            : rotary_kernel<T, L, true, false, TAIL, N><<<grid, kWarps * 32, 0, st>>>(a, per))
    if (!fast) rotary_any_kernel<T><<<grid, kWarps * 32, 0, st>>>(a, per);
    else if (wide) QMM_ROTARY(kWide);
    else if (a.adjacent) QMM_ROTARY(kAdjacent);
    else QMM_ROTARY(kHalves);
#undef QMM_ROTARY_T
#undef QMM_ROTARY_N
#undef QMM_ROTARY
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? QMM_OK : cuda_fail(e, "rotary launch");
}

}  // namespace rotary
}  // namespace qmm

using qmm::fail;

namespace {

struct Span {
    uintptr_t lo, hi;
};
// Bytes from the first to the last element of [batch, tokens, heads, dim] at the given strides (none negative).
Span span_of(const void *p, const qmm_rotary_args &a, int heads, const int64_t *stride, int64_t esize) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(p);
    const int64_t last = (a.batch - 1) * stride[0] + (a.tokens - 1) * stride[1] + (heads - 1) * stride[2] + a.dim;
    return Span{b, b + (uintptr_t)(last * esize)};
}
bool overlap(const Span &a, const Span &b) { return a.lo < b.hi && b.lo < a.hi; }
bool same_strides(const int64_t *a, const int64_t *b) { return a[0] == b[0] && a[1] == b[1] && a[2] == b[2]; }

// Whether some two heads of [batch, tokens, heads] share an element: each dimension's stride must reach past the
// extent of those with smaller strides.
bool self_overlap(const qmm_rotary_args &a, int heads, const int64_t *stride) {
    struct D {
        int64_t n, s;
    } d[3] = {{a.batch, stride[0]}, {a.tokens, stride[1]}, {heads, stride[2]}};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (d[j].s < d[i].s) {
                const D t = d[i];
                d[i] = d[j];
                d[j] = t;
            }
    int64_t extent = a.dim;
    for (const D &x : d) {
        if (x.n <= 1) continue;
        if (x.s < extent) return true;
        extent += (x.n - 1) * x.s;
    }
    return false;
}

// Whether two operands are certain to share no element: apart in memory, or side by side inside one buffer (a fused
// projection): the same batch and token strides and, within a token, one after the other or alternating head by head.
bool apart(const qmm_rotary_args &a, const void *p, int ph, const int64_t *ps, const void *q, int qh, const int64_t *qs, int64_t esize) {
    if (!overlap(span_of(p, a, ph, ps, esize), span_of(q, a, qh, qs, esize))) return true;
    if (ps[0] != qs[0] || ps[1] != qs[1] || self_overlap(a, ph, ps) || self_overlap(a, qh, qs)) return false;
    if (reinterpret_cast<uintptr_t>(p) > reinterpret_cast<uintptr_t>(q)) return apart(a, q, qh, qs, p, ph, ps, esize);
    const int64_t bytes = (int64_t)(reinterpret_cast<uintptr_t>(q) - reinterpret_cast<uintptr_t>(p));
    if (bytes % esize) return false;
    const int64_t d = bytes / esize, pe = (ph - 1) * ps[2] + a.dim, qe = (qh - 1) * qs[2] + a.dim;
    // the smallest stride that separates two tokens (or batches) of an operand
    int64_t period = INT64_MAX;
    if (a.tokens > 1 && ps[1] < period) period = ps[1];
    if (a.batch > 1 && ps[0] < period) period = ps[0];
    if (d >= pe && d + qe <= period) return true;
    const int64_t most = ph > qh ? ph : qh;
    return ps[2] == qs[2] && d >= a.dim && d + a.dim <= ps[2] && (most - 1) * ps[2] + d + a.dim <= period;
}

}  // namespace

extern "C" qmm_status qmm_qk_norm_rotary(const qmm_rotary_args *p, void *stream) {
    if (!p) return fail(QMM_ERR_INVALID_ARGUMENT, "rotary: null arguments");
    qmm_rotary_args a = *p;
    if (!a.k) a.k_heads = 0;
    if (a.batch < 0 || a.tokens < 0 || a.q_heads < 0 || a.k_heads < 0 || a.dim <= 0 || a.pairs < 0 || 2 * (int64_t)a.pairs > a.dim || a.axes <= 0 || a.axes > 256)
        return fail(QMM_ERR_BAD_SHAPE, "rotary: %lld x %lld tokens, %d and %d heads of %d, %d pairs over %d axes", (long long)a.batch,
                    (long long)a.tokens, a.q_heads, a.k_heads, a.dim, a.pairs, a.axes);
    if (a.dim > 256) return fail(QMM_ERR_UNSUPPORTED, "rotary: heads of %d columns (at most 256)", a.dim);
    if (a.elem < QMM_ELEM_BF16 || a.elem > QMM_ELEM_F16 || a.pos_kind < 0 || a.pos_kind > 2)
        return fail(QMM_ERR_INVALID_ARGUMENT, "rotary: element type %d, position type %d", a.elem, a.pos_kind);
    if (a.batch == 0 || a.tokens == 0 || a.q_heads + a.k_heads == 0) return QMM_OK;
    if ((a.q_heads && (!a.q || !a.q_out)) || (a.k_heads && !a.k_out)) return fail(QMM_ERR_INVALID_ARGUMENT, "rotary: null q, k or output");
    if (a.pairs && (!a.positions || !a.turns || !a.axis)) return fail(QMM_ERR_INVALID_ARGUMENT, "rotary: null positions, turns or axis");
    const int64_t esize = a.elem == QMM_ELEM_F32 ? 4 : 2;
    struct Operand {
        const void *src, *dst;
        const int64_t *ss, *ds;
        int heads;
    } const ops[2] = {{a.q, a.q_out, a.q_stride, a.q_out_stride, a.q_heads}, {a.k, a.k_out, a.k_stride, a.k_out_stride, a.k_heads}};
    for (const Operand &o : ops) {
        if (!o.heads) continue;
        for (int i = 0; i < 3; ++i)
            if (o.ss[i] < 0 || o.ds[i] < 0) return fail(QMM_ERR_BAD_SHAPE, "rotary: negative stride");
        if (reinterpret_cast<uintptr_t>(o.src) % esize || reinterpret_cast<uintptr_t>(o.dst) % esize)
            return fail(QMM_ERR_MISALIGNED, "rotary: a pointer is not aligned to its element");
        if (self_overlap(a, o.heads, o.ds)) return fail(QMM_ERR_BAD_SHAPE, "rotary: the output's strides make heads overlap");
    }
    // In place (each head is read whole before it is written) or apart.
    for (const Operand &o : ops) {
        if (!o.heads) continue;
        if (!(o.src == o.dst && same_strides(o.ss, o.ds)) && !apart(a, o.src, o.heads, o.ss, o.dst, o.heads, o.ds, esize))
            return fail(QMM_ERR_INVALID_ARGUMENT, "rotary: an output overlaps its input without being it");
    }
    if (a.q_heads && a.k_heads &&
        (!apart(a, a.q_out, a.q_heads, a.q_out_stride, a.k_out, a.k_heads, a.k_out_stride, esize) ||
         !apart(a, a.q_out, a.q_heads, a.q_out_stride, a.k, a.k_heads, a.k_stride, esize) ||
         !apart(a, a.k_out, a.k_heads, a.k_out_stride, a.q, a.q_heads, a.q_stride, esize)))
        return fail(QMM_ERR_INVALID_ARGUMENT, "rotary: an output overlaps the other operand");
    const int64_t wsize = esize;
    if (reinterpret_cast<uintptr_t>(a.q_weight) % wsize || reinterpret_cast<uintptr_t>(a.k_weight) % wsize ||
        reinterpret_cast<uintptr_t>(a.turns) % 4 || reinterpret_cast<uintptr_t>(a.positions) % (a.pos_kind == 1 ? 8 : 4))
        return fail(QMM_ERR_MISALIGNED, "rotary: weights, turns or positions are not aligned to their element");
    const qmm_status s = qmm::check_device();
    if (s != QMM_OK) return s;
    // fast: runs of four elements; wide: adjacent pairs, runs of eight (16 bytes of a 16-bit type)
    bool fast = a.dim % 8 == 0 && (a.adjacent || a.pairs % 4 == 0), wide = a.adjacent != 0;
    const uintptr_t quad = (uintptr_t)(4 * esize);
    auto judge = [&](const void *p, const int64_t *strides) {
        fast = fast && reinterpret_cast<uintptr_t>(p) % quad == 0;
        wide = wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
        for (int i = 0; strides && i < 3; ++i) {
            fast = fast && strides[i] % 4 == 0;
            wide = wide && (strides[i] * esize) % 16 == 0;
        }
    };
    for (const Operand &o : ops) {
        if (!o.heads) continue;
        judge(o.src, o.ss);
        judge(o.dst, o.ds);
    }
    judge(a.q_weight, nullptr);
    judge(a.k_weight, nullptr);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.elem == QMM_ELEM_F32) return qmm::rotary::launch<float>(a, fast, wide, st);
    if (a.elem == QMM_ELEM_F16) return qmm::rotary::launch<qmm::F16>(a, fast, wide, st);
    return qmm::rotary::launch<qmm::Bf16>(a, fast, wide, st);
}
