// MXFP4 product for few tokens:  y [m, n] = epilogue(x [m, k] . W [n, k]^T).
//
// With few tokens the time is the weight's way out of HBM, so the weight rows are the
// MMA's M: a CTA takes 128 features x NT tokens (N = 16 .. 128) and streams its rows'
// codes (17 KB a stage of 256 columns, scales included) through a ring that holds most
// or all of them at once.  Where the tiles do not fill the SMs, a cluster of CTAs
// splits k and sums its partial tiles over distributed shared memory, always in the
// same order.
//
// x needs no pass of its own: 16 warps quantise this CTA's columns of it while the
// weight is on its way (a warp a row of 256 columns: eight columns a lane, four lanes a
// block), writing codes and scales straight into the stage's operand layout; an x that
// is MXFP4 already comes by TMA instead.  The same warps then run the epilogue.
//
// HBM-bound where the weight is large, latency-bound where it is not.  B200, back to
// back: 1 x 3072 -> 18432 7.1 us (30 MB: 4.6 us of HBM, the rest is the launch, the first
// stage's arrival and the last tile's epilogue), 1 x 12288 -> 3072 7.6 us, 128 x 3072 ->
// 12288 10.7 us, 8 x 512 -> 512 3.5 us.
#include <algorithm>
#include <cstring>

#include "qmm_mx4_mma.cuh"

namespace qmm {
namespace mx4 {
namespace small {

constexpr int kRows = 128;  // features a tile
constexpr int kWorkers = 16;
constexpr int kProducer = kWorkers, kMma = kWorkers + 1;
constexpr int kThreads = (kWorkers + 2) * 32;
constexpr int kMaxSplit = 8;

template <int NT>
struct Cfg {
    static constexpr int kABytes = kRows * kRowBytes;
    static constexpr int kBBytes = NT * kRowBytes;
    static constexpr int kSfBytes = 2 * kSfTile;
    static constexpr int kStageBytes = kABytes + kBBytes + 2 * kSfBytes;
    static constexpr int kSfCols = 16;  // tensor-memory columns of a stage's scales: 8 for each operand
    static constexpr int kFit = (232448 - 1024 - 512) / kStageBytes;
    static constexpr int kSlots = (512 - NT) / kSfCols;
    static constexpr int kStages = kFit < kSlots ? (kFit < 12 ? kFit : 12) : kSlots;
    static constexpr int kTmemCols = NT + kStages * kSfCols <= 256 ? 256 : 512;
    static constexpr int kAOff = 0;
    static constexpr int kBOff = kAOff + kStages * kABytes;
    static constexpr int kSfaOff = kBOff + kStages * kBBytes;
    static constexpr int kSfbOff = kSfaOff + kStages * kSfBytes;
    static constexpr int kBarOff = kSfbOff + kStages * kSfBytes;
    static constexpr int kNumBars = 3 * kStages + 2;
    static constexpr int kSmemBytes = kBarOff + kNumBars * 8 + 16 + 1024;
    static_assert(kSmemBytes <= 232448 && kStages * kABytes >= NT * kRows * 4, "shared memory");
    static constexpr uint32_t kIdesc = idesc_mxf4(kRows, NT);
};

struct Params {
    const uint8_t *w_scales, *x_scales;
    const void *x;           // null: x is MXFP4 and comes by TMA
    int64_t x_row_stride;
    EpilogueArgs ep;
    uint16_t *y;
    int32_t m, n, k;
    int32_t nkb, sf_tiles;   // stages along k; scale tiles along k
    int32_t vec;             // rows of x on 16-byte boundaries, k a multiple of 8
    uint32_t *err;
};

__device__ __forceinline__ float4 load_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

template <int COLS>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[COLS]) {
    if constexpr (COLS == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(taddr));
    } else if constexpr (COLS == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
              "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
    } else {
        tmem_ld_32x32b_x32(taddr, r);
    }
}

// One value of y: feature f of token t.
__device__ __forceinline__ void finish(const Params &p, float acc, float bias, float gate, int64_t t, int64_t f) {
    float v = acc + bias;
    if (p.ep.act == QMM_ACT_GELU_TANH) v = activate<true>(make_float2(v, v)).x;
    else if (p.ep.act == QMM_ACT_SILU) v = activate<false>(make_float2(v, v)).x;
    v *= gate;
    if (p.ep.residual) {
        const float r = bf16_bits_to_f32(p.ep.residual[t * p.n + f]);
        v = p.ep.res_mul ? r * v : r + v;
    }
    p.y[t * p.n + f] = f32_to_bf16_bits(v);
}

// Grid (split, row tiles, token tiles), clusters of `split` CTAs along k.
template <typename T, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    mx4_small_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Params p) {
    using C = Cfg<NT>;
    constexpr int S = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::kBarOff);  // [S] copies landed
    uint64_t *xfull = full + S;                                        // [S] x rows quantised
    uint64_t *empty = xfull + S;                                       // [S] stage's MMAs complete
    uint64_t *acc_full = empty + S;
    uint64_t *drain = acc_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = gridDim.x, rank = blockIdx.x;
    const int n0 = blockIdx.y * kRows, m0 = blockIdx.z * NT;
    const int tokens = min(NT, p.m - m0);
    const int kb0 = p.nkb * rank / split, nkb = p.nkb * (rank + 1) / split - kb0;  // this CTA's stages (one at least)
    const bool quantise = p.x != nullptr;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&xfull[s], (uint32_t)tokens);
            mbar_init(&empty[s], 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(drain, 1);
        fence_barrier_init();
    }
    if (warp == kMma) {
        tmem_alloc(tmem_slot, C::kTmemCols);
        tmem_relinquish();
    }
    if (warp == kProducer && lane == 0) {
        tma_prefetch_desc(&tmap_w);
        if (!quantise) tma_prefetch_desc(&tmap_x);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == kProducer) {
        // ------------------------------------------------------------ copies
        auto copy_weight = [&](int i) {
            const int s = i % S;
            mbar_arrive_expect_tx(&full[s], C::kABytes + C::kSfBytes + (quantise ? 0 : C::kBBytes + C::kSfBytes));
            tma_load_2d(smem + C::kAOff + s * C::kABytes, &tmap_w, &full[s], (kb0 + i) * kRowBytes, n0);
            bulk_load(smem + C::kSfaOff + s * C::kSfBytes, p.w_scales + ((int64_t)(n0 >> 7) * p.sf_tiles + (kb0 + i) * 2) * kSfTile,
                      C::kSfBytes, &full[s]);
        };
        auto copy_x = [&](int i) {
            const int s = i % S;
            tma_load_2d(smem + C::kBOff + s * C::kBBytes, &tmap_x, &full[s], (kb0 + i) * kRowBytes, m0);
            // (m0 is a multiple of 128: tiles of fewer tokens come alone)
            bulk_load(smem + C::kSfbOff + s * C::kSfBytes, p.x_scales + ((int64_t)(m0 >> 7) * p.sf_tiles + (kb0 + i) * 2) * kSfTile,
                      C::kSfBytes, &full[s]);
        };
        const int first = min(S, nkb);
        // The weight too: the kernel ahead may be the quantisation that makes it.
        pdl_dependency_wait();
        if (lane == 0) {
            for (int i = 0; i < first; ++i) {
                copy_weight(i);
                if (!quantise) copy_x(i);
            }
        }
        __syncwarp();
        int i = first;
        for (; i < nkb; ++i) {
            if (!mbar_wait(&empty[i % S], ((i / S) & 1) ^ 1, p.err, kErrTimeoutProducer)) {
                ok = false;
                break;
            }
            if (lane == 0) {
                copy_weight(i);
                if (!quantise) copy_x(i);
            }
            __syncwarp();
        }
        pdl_launch_dependents();
        if (!ok)  // let the copies already issued land before the CTA exits
            for (int j = max(0, i - S); j < i; ++j) mbar_wait(&full[j % S], (j / S) & 1, p.err, kErrTimeoutDrain);
    } else if (warp == kMma) {
        // ------------------------------------------------------------ MMA issuer
        const uint64_t adesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kAOff)), bdesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kBOff));
        const uint64_t sadesc0 = sdesc_scales(smem_u32(smem + C::kSfaOff)), sbdesc0 = sdesc_scales(smem_u32(smem + C::kSfbOff));
        uint32_t acc = 0;
        int i = 0;
        for (; i < nkb; ++i) {
            const int s = i % S;
            ok = mbar_wait(&full[s], (i / S) & 1, p.err, kErrTimeoutMma);
            if (ok && quantise) ok = mbar_wait(&xfull[s], (i / S) & 1, p.err, kErrTimeoutMma);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after_sync();
            if (lane_elect()) {
                const uint32_t sfa = tmem + NT + s * C::kSfCols, sfb = sfa + 8;
                const uint64_t ad = adesc0 + (uint64_t)s * (C::kABytes >> 4), bd = bdesc0 + (uint64_t)s * (C::kBBytes >> 4);
                const uint64_t sad = sadesc0 + (uint64_t)s * (C::kSfBytes >> 4), sbd = sbdesc0 + (uint64_t)s * (C::kSfBytes >> 4);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    tc_copy_scales(sfa + h * 4, sad + h * (kSfTile >> 4));
                    tc_copy_scales(sfb + h * 4, sbd + h * (kSfTile >> 4));
                }
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    tc_mma_mxf4(tmem, ad + kk * 2, bd + kk * 2, C::kIdesc | idesc_scale_id((kk & 1) * 2), sfa + (kk >> 1) * 4,
                                sfb + (kk >> 1) * 4, acc);
                    acc = 1;
                }
                tc_commit(&empty[s]);
                if (i + 1 == nkb) tc_commit(acc_full);
            }
            acc = 1;
            __syncwarp();
        }
        if (!ok && i > 0) {
            if (lane_elect()) tc_commit(drain);
            __syncwarp();
            mbar_wait(drain, 0, p.err, kErrTimeoutDrain);
        }
    } else {
        pdl_dependency_wait();
        if (quantise) {
            // -------------------------------------------------------- x to MXFP4
            // A warp's units of each turn of the ring are (slot, row) pairs kWorkers apart, the same ones in every turn: so it
            // has seen each of its slots' phases, and the parity that it waits for is never two phases away.
            const T *const x = static_cast<const T *>(p.x) + (int64_t)m0 * p.x_row_stride;
            constexpr int kFlight = sizeof(T) == 4 ? 4 : 8;  // units whose loads a warp has in flight
            auto fetch = [&](int i, int r) {
                const int64_t c = (int64_t)(kb0 + i) * kBK + lane * 8;
                const T *const src = x + (int64_t)r * p.x_row_stride + c;
                Vec8<T> raw{};
                if (p.vec) {
                    if (c < p.k) raw = load_vec8(src);
                } else {
                    T e[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        e[j] = T{};
                        if (c + j < p.k) e[j] = src[j];
                    }
                    memcpy(&raw, e, sizeof raw);
                }
                return raw;
            };
            for (int turn = 0; ok && turn * S < nkb; ++turn) {
                const int units = min(S, nkb - turn * S) * tokens;
                for (int u0 = warp; ok && u0 < units; u0 += kFlight * kWorkers) {
                    Vec8<T> raw[kFlight];
#pragma unroll
                    for (int j = 0; j < kFlight; ++j) {
                        const int u = u0 + j * kWorkers, s = u / tokens;
                        if (u < units) raw[j] = fetch(turn * S + s, u - s * tokens);
                    }
#pragma unroll
                    for (int j = 0; j < kFlight; ++j) {
                        const int u = u0 + j * kWorkers, s = u / tokens, r = u - s * tokens;
                        if (!ok || u >= units) break;
                        if (turn > 0) {  // the MMAs of the turn before have read the slot
                            ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (turn & 1) ^ 1, p.err, kErrTimeoutDequant));
                            if (!ok) break;
                        }
                        float v[8];
                        vec8_to_f32(raw[j], v);
                        uint32_t codes;
                        const uint32_t e = mx4_encode8(v, &codes);
                        uint32_t word = e << (8 * ((lane >> 2) & 3));
                        word |= __shfl_xor_sync(0xffffffffu, word, 4);
                        word |= __shfl_xor_sync(0xffffffffu, word, 8);
                        // 16-byte cells of a 128-byte row are swizzled by the row's place in eight
                        *reinterpret_cast<uint32_t *>(smem + C::kBOff + s * C::kBBytes + r * kRowBytes + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = codes;
                        if ((lane & 15) == 0)
                            *reinterpret_cast<uint32_t *>(smem + C::kSfbOff + s * C::kSfBytes + (lane >> 4) * kSfTile + (r & 31) * 16 + (r >> 5) * 4) = word;
                    }
                    // one fence for the batch, then its rows are announced
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (ok && lane == 0)
                        for (int u = u0; u < min(u0 + kFlight * kWorkers, units); u += kWorkers) mbar_arrive(&xfull[u / tokens]);
                }
            }
        }
        // ------------------------------------------------------------ epilogue
        const int quad = warp & 3, group = warp >> 2;
        const int64_t f = n0 + quad * 32 + lane;
        const FeatureConsts fc = load_feature_consts(p.ep, f, f < p.n);
        ok = ok && __all_sync(0xffffffffu, mbar_wait(acc_full, 0, p.err, kErrTimeoutEpilogue));
        if (ok) {
            tc_fence_after_sync();
            constexpr int kCols = NT / 4 < 8 ? 8 : NT / 4;  // tokens a warp (16: two of the four groups)
            float *const part = reinterpret_cast<float *>(smem + C::kAOff);  // [NT][kRows]: every MMA on the ring is complete
            const int t0 = group * kCols;
            if (t0 < tokens) {
                uint32_t r[kCols];
                tmem_ld(tmem + ((uint32_t)(quad * 32) << 16) + t0, r);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    if (t0 + c < tokens) {
                        if (split > 1) part[(t0 + c) * kRows + quad * 32 + lane] = __uint_as_float(r[c]);
                        else if (f < p.n) finish(p, __uint_as_float(r[c]), fc.bias, fc.gate, m0 + t0 + c, f);
                    }
                }
            }
        }
    }
    tc_fence_before_sync();
    if (split == 1) {
        __syncthreads();
    } else {
        // Each CTA of the cluster sums every `split`-th token's partial tiles, in the order of k.  (After an expired wait
        // anywhere the sums are of no use, as the error word says.)
        __syncthreads();
        cluster_sync();
        if (warp < kWorkers) {  // a warp a token, four features a lane
            const int64_t f = n0 + lane * 4;
            FeatureConsts fc[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) fc[i] = load_feature_consts(p.ep, f + i, f + i < p.n);
            const uint32_t part = smem_u32(smem + C::kAOff) + lane * 16;
            for (int t = rank + split * warp; t < tokens; t += split * kWorkers) {
                float4 v[kMaxSplit];
#pragma unroll
                for (int j = 0; j < kMaxSplit; ++j) v[j] = j < split ? load_cluster_f32x4(mapa_shared(part + t * kRows * 4, j)) : float4{};
                float4 s = v[0];
#pragma unroll
                for (int j = 1; j < kMaxSplit; ++j) s.x += v[j].x, s.y += v[j].y, s.z += v[j].z, s.w += v[j].w;
                if (f < p.n) finish(p, s.x, fc[0].bias, fc[0].gate, m0 + t, f);
                if (f + 1 < p.n) finish(p, s.y, fc[1].bias, fc[1].gate, m0 + t, f + 1);
                if (f + 2 < p.n) finish(p, s.z, fc[2].bias, fc[2].gate, m0 + t, f + 2);
                if (f + 3 < p.n) finish(p, s.w, fc[3].bias, fc[3].gate, m0 + t, f + 3);
            }
        }
        cluster_sync();  // no CTA leaves while another reads its partial tile
    }
    if (warp == kMma) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, C::kTmemCols);
    }
}

template <typename T, int NT>
static qmm_status launch(const qmm_mx4 &w, const void *x, int64_t x_row_stride, const qmm_mx4 &xq, const qmm_epilogue &ep, uint16_t *y, int split,
                         cudaStream_t st) {
    using C = Cfg<NT>;
    static bool configured[64] = {};
    qmm_status s = allow_smem(mx4_small_kernel<T, NT>, C::kSmemBytes, configured);
    if (s != QMM_OK) return s;
    const uint64_t pitch = (uint64_t)mx4_pitch(w.k);
    CUtensorMap tw, tx;
    s = map_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes, pitch, (uint64_t)w.rows, pitch, kRowBytes, kRows, CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != QMM_OK) return s;
    tx = tw;
    if (!x) s = map_2d(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, xq.codes, pitch, (uint64_t)xq.rows, pitch, kRowBytes, NT, CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != QMM_OK) return s;
    Params p;
    p.w_scales = w.scales;
    p.x_scales = xq.scales;
    p.x = x;
    p.x_row_stride = x_row_stride;
    p.ep = epilogue_args(ep);
    p.y = y;
    p.m = (int32_t)xq.rows;
    p.n = (int32_t)w.rows;
    p.k = (int32_t)w.k;
    p.nkb = (int32_t)((w.k + kBK - 1) / kBK);
    p.sf_tiles = (int32_t)mx4_scale_tiles(w.k);
    p.vec = w.k % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (xq.rows == 1 || (x_row_stride * (int64_t)sizeof(T)) % 16 == 0);
    p.err = device_error_word();
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3((unsigned)split, (unsigned)((w.rows + kRows - 1) / kRows), (unsigned)((xq.rows + NT - 1) / NT));
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, mx4_small_kernel<T, NT>, tw, tx, p);
    count_launch();
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? QMM_OK : cuda_fail(e, "mxfp4 product launch");
}

// CTAs along k: as many as keep the grid within `sms`, where that takes eight stages
// or more out of a CTA's way: a stage costs 0.24 us, the cluster's sum about 1.2 us
// (B200, one token: 12288 -> 3072 7.6 us split against 15.3, 3072 -> 3072 4.8 against
// 5.2; 3072 -> 9216 in two 6.2 against 5.8).
static int split_for(int64_t tiles, int64_t nkb, int sms) {
    int split = 1;
    while (split < kMaxSplit && split * 2 <= nkb && tiles * split * 2 <= sms) split *= 2;
    return nkb - (nkb + split - 1) / split >= 8 ? split : 1;
}

// Tokens a tile for m tokens, and the tiles.
static int tile_for(int64_t m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128; }
static int64_t tiles_for(const qmm_mx4 &w, int64_t m) {
    const int nt = tile_for(m);
    return (w.rows + kRows - 1) / kRows * ((m + nt - 1) / nt);
}

}  // namespace small

// The rules below count the SMs of a B200, not those left by an SM budget: what a
// call needs does not change between asking for its workspace and making it.
constexpr int kSms = 148;

bool mx4_small_fits(int64_t n, int64_t m) {
    // Up to one tile of tokens, or where the 128 x 192 tiles of the other kernel
    // would leave half of the SMs idle.
    if ((n + small::kRows - 1) / small::kRows > 65535 || (m + 127) / 128 > 65535) return false;
    return m <= 128 || (m + 127) / 128 * ((n + 191) / 192) * 2 < kSms;
}

bool mx4_small_quantises(int64_t n, int64_t m, int64_t k) {
    // Every tile of features quantises its columns of x for itself.  Up to six rows of
    // a stage a warp a call is shorter that way than with a pass over x before it (B200,
    // 8 x 3072 -> 9216, six a warp: 9.7 us against 10.3; 37 x 1152 -> 3456, twelve: 11.2
    // against 9.3).
    const qmm_mx4 w{nullptr, nullptr, n, k};
    const int64_t nkb = (k + kBK - 1) / kBK, split = small::split_for(small::tiles_for(w, m), nkb, kSms);
    return (nkb + split - 1) / split * std::min<int64_t>(m, small::tile_for(m)) <= 6 * small::kWorkers;
}

qmm_status launch_mx4_small(const qmm_mx4 &w, const void *x, int32_t elem, int64_t x_row_stride, const qmm_mx4 &xq, const qmm_epilogue &ep,
                            uint16_t *y, cudaStream_t st) {
    const int nt = small::tile_for(xq.rows);
    const int split = small::split_for(small::tiles_for(w, xq.rows), (w.k + kBK - 1) / kBK, sm_count());
#define QMM_MX4_SMALL(T)                                                                                    \
    (nt == 16   ? small::launch<T, 16>(w, x, x_row_stride, xq, ep, y, split, st)                            \
     : nt == 32 ? small::launch<T, 32>(w, x, x_row_stride, xq, ep, y, split, st)                            \
     : nt == 64 ? small::launch<T, 64>(w, x, x_row_stride, xq, ep, y, split, st)                            \
                : small::launch<T, 128>(w, x, x_row_stride, xq, ep, y, split, st))
    if (!x || elem == QMM_ELEM_BF16) return QMM_MX4_SMALL(Bf16);
    return elem == QMM_ELEM_F16 ? QMM_MX4_SMALL(F16) : QMM_MX4_SMALL(float);
#undef QMM_MX4_SMALL
}

}  // namespace mx4
}  // namespace qmm
