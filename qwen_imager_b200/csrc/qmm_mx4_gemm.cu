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
// Warp roles (one persistent CTA per SM): 12 epilogue warps (three per lane quadrant,
// two chunks of 32 columns each; 16 share them no better and leave 96 registers a
// thread instead of 128: 16384 x 256 -> 12288 115 us against 96), a producer warp (TMA for
// codes, bulk copies for scales), an MMA warp (one elected lane issues copies, MMAs and commits).  Two
// accumulators, so a tile's epilogue overlaps the next tile's main loop.  Scale
// slots in tensor memory are tied to the shared-memory stages: a stage refilled
// means that the MMAs that read its slot are complete.  Every wait is bounded.
//
// Bounds (B200): with k short the epilogue (16384 x 256 -> 12288 96 us, 4.2 TB/s of y;
// with GELU 163, its exponentials and reciprocals); with k long the loads, 43 KB a
// stage (4352 x 12288 -> 3072 77 us, 57 on pairs, below).
#include <algorithm>
#include <climits>

#include "qmm_mx4_mma.cuh"

namespace qmm {
namespace mx4 {

constexpr int kTM = 128;         // tokens a tile
constexpr int kChunk = 32;       // columns an epilogue step

// A CTA's warps: EPI for the epilogue, then the producer and the MMA issuer.
template <int EPI, int CHUNKS>
struct Warps {
    static constexpr int kMaxChunks = CHUNKS;  // of an epilogue warp in a tile
    static constexpr int kEpiWarps = EPI, kProducer = EPI, kMma = EPI + 1, kThreads = (EPI + 2) * 32;
    static constexpr int kGroups = EPI / 4;  // epilogue warps on each lane quadrant: chunk c is group c % kGroups
};

template <int TN>
struct Cfg : Warps<12, 2> {
    using W = Warps<12, 2>;
    static_assert(TN % 64 == 0 && TN <= 256, "feature tile");
    static constexpr int kABytes = kTM * kRowBytes;
    static constexpr int kBBytes = TN * kRowBytes;
    static constexpr int kBTiles = (TN + 127) / 128;  // 128-row scale tiles under B; a start at row 64 of one still fits
    static constexpr int kSfaBytes = 2 * kSfTile;
    static constexpr int kSfbBytes = 2 * kBTiles * kSfTile;
    static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
    static constexpr int kOutBytes = W::kEpiWarps * kChunk * 64;  // a 32 x 32 bf16 buffer a warp
    static constexpr int kVecBytes = W::kEpiWarps * W::kMaxChunks * 2 * kChunk * 4;  // bias and gate of a warp's chunks
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
    static constexpr int kNumBars = 2 * kStages + 4 + 1 + W::kEpiWarps;
    static constexpr int kSmemBytes = kBarOff + kNumBars * 8 + 16 + 1024;
    static constexpr int kSfCol0 = 2 * TN;
    static_assert(kStages >= 2 && kSmemBytes <= 232448, "shared memory");
    static constexpr uint32_t kIdesc = idesc_mxf4(kTM, TN);
};

struct Params {
    const uint8_t *a_scales, *b_scales;
    EpilogueArgs ep;
    uint16_t *y;
    int32_t m, n;
    int32_t nkb, sf_tiles;       // stages along k; scale tiles along k
    int32_t m_tiles, n_tiles;
    int32_t b_row_tiles;         // 128-row scale tiles of W
    uint32_t *err;
};

// Tile t of the persistent loop.  (Patches of 4, 8 and 16 tiles of tokens measured the same.)
__device__ __forceinline__ void tile_at(const Params &p, int t, int &mt, int &nt) {
    nt = t / p.m_tiles;
    mt = t - nt * p.m_tiles;
}

// What an epilogue warp owns in shared memory.
struct ChunkOut {
    uint8_t *stage;     // 32 tokens x 32 features of bf16: 64 bytes a token, 16-byte cells swizzled
    float *vec;         // bias[32], gate[32] of each of the tile's chunks
    uint64_t *res_full; // a residual chunk landed in `stage`
};

__device__ __forceinline__ void request_residual(const CUtensorMap *tmap_res, const ChunkOut &o, int f0, int m0) {
    if ((threadIdx.x & 31) == 0) {
        bulk_wait_read<0>();  // the last store has left the buffer
        mbar_arrive_expect_tx(o.res_full, kChunk * 64);
        tma_load_2d(o.stage, tmap_res, o.res_full, f0, m0);
    }
}

// 32 tokens x 32 features in a warp's staging buffer, and their rows in global memory
// off 16-byte boundaries, which move by aligned 4-byte words, half a warp a token.
// Where a token's first feature is the upper half of a word (odd), its cells hold the
// words one feature earlier, and the last word is the lane's own (`behind`).  A lane's
// tokens are two apart, so the words it moves are of odd tokens or of none.
struct WordRows {
    uint8_t *stage;
    int64_t own;         // element of token `lane`
    int64_t first;       // element in the lower half of the lane's first word
    int nf, nt, f;       // features and tokens here; the feature of `first`
    __device__ __forceinline__ WordRows(const Params &p, uint8_t *buffer, int f0, int m0) : stage(buffer) {
        const int lane = threadIdx.x & 31, side = lane >> 4;
        nf = min(kChunk, p.n - f0), nt = min(32, p.m - m0);
        own = (int64_t)(m0 + lane) * p.n + f0;
        const int64_t e = (int64_t)(m0 + side) * p.n + f0;
        f = 2 * (lane & 15) - (int)(e & 1);
        first = e + f;
    }
    __device__ __forceinline__ bool odd() const { return own & 1; }
    __device__ __forceinline__ uint4 *cell(int g) const {
        const int lane = threadIdx.x & 31;
        return reinterpret_cast<uint4 *>(stage + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4));
    }
    // The lane's word of token t0 + 2 u + lane / 16, t0 a multiple of 8.
    __device__ __forceinline__ uint32_t *word(int t0, int u) const {
        const int lane = threadIdx.x & 31;
        return reinterpret_cast<uint32_t *>(stage + (t0 + 2 * u + (lane >> 4)) * 64 + ((((lane & 15) >> 2) ^ (u & 3)) << 4) + (lane & 3) * 4);
    }
    __device__ __forceinline__ void load(const uint16_t *p, int n) const {
        const int lane = threadIdx.x & 31;
        uint32_t behind = 0;
        if (odd() && lane < nt && nf == kChunk) behind = p[own + kChunk - 1];
        const uint16_t *from = p + first;
        const int tokens = f < nf ? nt - (lane >> 4) : 0;
#pragma unroll 1
        for (int t0 = 0; t0 < 32; t0 += 16) {
            uint32_t w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                w[u] = 0;
                if (t0 + 2 * u < tokens) {  // (before the first feature: the token before's last; past the last: not read)
                    if (f + 1 < nf) w[u] = *reinterpret_cast<const uint32_t *>(from);
                    else w[u] = *from;
                }
                from += 2 * (int64_t)n;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) *word(t0, u) = w[u];
        }
        __syncwarp();
        if (odd()) {
            uint4 c[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) c[g] = *cell(g);
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *cell(g) = make_uint4(__funnelshift_r(c[g].x, c[g].y, 16), __funnelshift_r(c[g].y, c[g].z, 16), __funnelshift_r(c[g].z, c[g].w, 16),
                                      __funnelshift_r(c[g].w, g < 3 ? c[(g + 1) & 3].x : behind, 16));
        }
    }
    // w: the lane's token.
    __device__ __forceinline__ void store(uint16_t *y, int n, uint32_t (&w)[16]) const {
        const int lane = threadIdx.x & 31;
        const uint32_t behind = w[15] >> 16;
        if (odd()) {
#pragma unroll
            for (int i = 15; i >= 0; --i) w[i] = __funnelshift_l(i ? w[i > 0 ? i - 1 : 0] : 0u, w[i], 16);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) *cell(g) = make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
        if (lane < nt) {  // a token's first and last feature, where they are half a word
            if (odd()) y[own] = (uint16_t)(w[0] >> 16);
            if ((nf + odd()) & 1) {
                const int last = (nf - 1 + odd()) >> 1;
                const uint32_t *const c = reinterpret_cast<const uint32_t *>(cell((last & 15) >> 2)) + (last & 3);
                y[own + nf - 1] = (uint16_t)(last < 16 ? *c : behind);
            }
        }
        __syncwarp();
        uint16_t *to = y + first;
        const int tokens = f >= 0 && f + 1 < nf ? nt - (lane >> 4) : 0;
#pragma unroll 1
        for (int t0 = 0; t0 < 32; t0 += 8) {
            uint32_t c[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) c[u] = *word(t0, u);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (t0 + 2 * u < tokens) *reinterpret_cast<uint32_t *>(to) = c[u];
                to += 2 * (int64_t)n;
            }
        }
        __syncwarp();
    }
};

// One warp's 32 tokens x 32 features, from the accumulators in r (a token a lane)
// through its staging buffer to y.  TMA: rows of y and the residual lie on 16-byte
// boundaries and move by TMA; the residual is in the buffer already.
template <bool TMA>
__device__ __forceinline__ void chunk_finish(const Params &p, const CUtensorMap *tmap_y, const ChunkOut &o, const float *vec, uint32_t (&r)[32],
                                             int f0, int m0) {
    const int lane = threadIdx.x & 31;
    const float4 *const bias = reinterpret_cast<const float4 *>(vec), *const gate = bias + kChunk / 4;
    // Each step over all 32 features: its branch is taken once, and the exponentials overlap.
    float v[32];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 b4 = bias[i];
        v[4 * i] = __uint_as_float(r[4 * i]) + b4.x;
        v[4 * i + 1] = __uint_as_float(r[4 * i + 1]) + b4.y;
        v[4 * i + 2] = __uint_as_float(r[4 * i + 2]) + b4.z;
        v[4 * i + 3] = __uint_as_float(r[4 * i + 3]) + b4.w;
    }
    if (p.ep.act == QMM_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float2 t = activate<true>(make_float2(v[i], v[i + 1]));
            v[i] = t.x, v[i + 1] = t.y;
        }
    } else if (p.ep.act == QMM_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float2 t = activate<false>(make_float2(v[i], v[i + 1]));
            v[i] = t.x, v[i + 1] = t.y;
        }
    }
    if (p.ep.gate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 g4 = gate[i];
            v[4 * i] *= g4.x;
            v[4 * i + 1] *= g4.y;
            v[4 * i + 2] *= g4.z;
            v[4 * i + 3] *= g4.w;
        }
    }
    auto cell = [&](int g) { return reinterpret_cast<uint4 *>(o.stage + lane * 64 + ((g ^ ((lane >> 1) & 3)) << 4)); };
    [[maybe_unused]] const WordRows rows(p, o.stage, f0, m0);
    if constexpr (!TMA) {
        if (p.ep.residual) rows.load(p.ep.residual, p.n);
    }
    if (p.ep.residual) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {  // eight features: 16 bytes of this token's row
            float res[8];
            Vec8<Bf16> w;
            w.w[0] = *cell(g);
            vec8_to_f32(w, res);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[g * 8 + e] = p.ep.res_mul ? res[e] * v[g * 8 + e] : res[e] + v[g * 8 + e];
        }
    }
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2_rn(v[2 * i], v[2 * i + 1]);
    if constexpr (TMA) {
        if (!p.ep.residual) {
            if (lane == 0) bulk_wait_read<0>();  // the last store has left the buffer
            __syncwarp();
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) *cell(g) = make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(tmap_y, o.stage, f0, m0);
            bulk_commit();
        }
    } else {
        rows.store(p.y, p.n, w);
    }
}

// A tile's chunks of one warp.  feature(c): the c-th chunk's first feature (p.n or more: none); column(c): its accumulator
// column; loaded(c) runs once chunk c is in registers; q counts the warp's chunks so far.  False: a wait ran out.
template <bool CLUSTER, bool TMA, int kMaxChunks, typename Feature, typename Column, typename Loaded>
__device__ __forceinline__ bool tile_epilogue(const Params &p, const CUtensorMap *tmap_y, const CUtensorMap *tmap_res, const ChunkOut &o, uint64_t *acc_full,
                                              uint32_t parity, uint32_t tmem, int m0, uint32_t &q, const Feature &feature, const Column &column,
                                              const Loaded &loaded) {
    const int lane = threadIdx.x & 31;
    const bool res_tma = TMA && p.ep.residual;
    // A quadrant past the last token or a chunk past the last feature has nothing to store.
    auto live = [&](int c) { return m0 < p.m && feature(c) < p.n; };
    bool requested = res_tma && live(0);
    if (requested) request_residual(tmap_res, o, feature(0), m0);
    {
        FeatureConsts fc[kMaxChunks];
#pragma unroll
        for (int c = 0; c < kMaxChunks; ++c) fc[c] = load_feature_consts(p.ep, feature(c) + lane, feature(c) + lane < p.n);
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kMaxChunks; ++c) {
            o.vec[c * 2 * kChunk + lane] = fc[c].bias;
            o.vec[c * 2 * kChunk + kChunk + lane] = fc[c].gate;
        }
        __syncwarp();
    }
    if (!__all_sync(0xffffffffu, mbar_wait<CLUSTER>(acc_full, parity, p.err, kErrTimeoutEpilogue))) {
        if (requested) mbar_wait(o.res_full, q & 1, p.err, kErrTimeoutDrain);
        return false;
    }
    tc_fence_after_sync();
#pragma unroll
    for (int c = 0; c < kMaxChunks; ++c) {
        uint32_t r[32];
        if (live(c)) {
            tmem_ld_32x32b_x32(tmem + column(c), r);
            if (res_tma && !requested) request_residual(tmap_res, o, feature(c), m0);
            tc_wait_ld();
        }
        loaded(c);
        if (live(c)) {
            if (res_tma && !__all_sync(0xffffffffu, mbar_wait(o.res_full, q & 1, p.err, kErrTimeoutEpilogue))) return false;
            chunk_finish<TMA>(p, tmap_y, o, o.vec + c * 2 * kChunk, r, feature(c), m0);
            requested = false;
            ++q;
        }
    }
    return true;
}

template <int TN, bool TMA>
__global__ void __launch_bounds__(Cfg<TN>::kThreads, 1)
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
    uint64_t *res_full = drain + 1;                                    // [warp] residual chunk landed
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(res_full + C::kEpiWarps);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], C::kEpiWarps);
        }
        mbar_init(drain, 1);
        for (int i = 0; i < C::kEpiWarps; ++i) mbar_init(&res_full[i], 1);
        fence_barrier_init();
    }
    if (warp == C::kMma) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == C::kProducer && lane == 0) {
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
        if (TMA) tma_prefetch_desc(&tmap_y);
        if (TMA && p.ep.residual) tma_prefetch_desc(&tmap_res);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const int tiles = p.m_tiles * p.n_tiles;

    if (warp == C::kProducer) {
        // ------------------------------------------------------------ producer
        pdl_dependency_wait();
        uint32_t i = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            int mt, nt;
            tile_at(p, t, mt, nt);
            const int m0 = mt * kTM, n0 = nt * TN;
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
    } else if (warp == C::kMma) {
        // ------------------------------------------------------------ MMA issuer
        bool ok = true, issued = false;
        uint32_t i = 0;
        int lt = 0;
        const uint64_t adesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kAOff)), bdesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kBOff));
        const uint64_t sadesc0 = sdesc_scales(smem_u32(smem + C::kSfaOff)), sbdesc0 = sdesc_scales(smem_u32(smem + C::kSfbOff));
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++lt) {
            int mt, nt;
            tile_at(p, t, mt, nt);
            const int n0 = nt * TN;
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
                        const uint32_t id = idesc_scale_id((kk & 1) * 2);
                        tc_mma_mxf4(d, ad + kk * 2, bd + kk * 2, C::kIdesc | id, sfa + (kk >> 1) * 4,
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
        const int quad = warp & 3, group = warp >> 2;
        const ChunkOut o{smem + C::kOutOff + warp * kChunk * 64, reinterpret_cast<float *>(smem + C::kVecOff) + warp * C::kMaxChunks * 2 * kChunk,
                         res_full + warp};
        uint32_t q = 0;
        int lt = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++lt) {
            int mt, nt;
            tile_at(p, t, mt, nt);
            const int m0 = mt * kTM + quad * 32, n0 = nt * TN;
            const int b = lt & 1;
            auto place = [&](int c) { return kChunk * (C::kGroups * c + group); };
            auto feature = [&](int c) { return place(c) < TN ? n0 + place(c) : INT_MAX - kChunk; };
            auto column = [&](int c) { return ((uint32_t)(quad * 32) << 16) + b * TN + place(c); };
            auto loaded = [&](int c) {
                if (c + 1 < C::kMaxChunks) return;
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[b]);
            };
            if (!tile_epilogue<false, TMA, C::kMaxChunks>(p, &tmap_y, &tmap_res, o, &acc_full[b], (lt >> 1) & 1, tmem, m0, q, feature, column, loaded)) break;
        }
        if (lane == 0) bulk_wait_all();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == C::kMma) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------- CTA pairs
// The same product on pairs of CTAs (cta_group::2): a tile of 256 tokens x 256
// features, each CTA holding 128 tokens and half of the features in its shared
// memory and accumulating its tokens for all of them.  Against the 128 x 192 tile
// of one CTA this reads 35 KB instead of 43 KB of operands for 1.33 times the
// work, and spreads six scale copies over it.  B200, back to back: 4352 x 12288 ->
// 3072 57 us (5.8 PFLOP/s; one-CTA tiles 77), 16384 x 3072 -> 12288 257 us, with GELU
// 277 (309, 332), without the epilogue's work 220: operands out of L2 and the power
// that all of it costs bound it (59, 265 and 289 in bursts of 100 launches on another
// card; after half a second the power cap leaves 1.6 GHz, 66, 295 and 323).  16 epilogue
// warps of 96 registers took 291 with GELU.
//
// Two accumulators of 256 columns and a scale slot for each stage do not fit the
// 512 columns of tensor memory, so the accumulators share 96 columns, [0, 256) and
// [160, 416), and four scale slots serve five stages.  The epilogue takes the chunks
// that hold the shared columns first, and the next tile's main loop starts once they
// are in registers.
struct PairCfg : Warps<12, 3> {
    static constexpr int kTN = 256;
    static constexpr int kABytes = kTM * kRowBytes;
    static constexpr int kBBytes = kTN / 2 * kRowBytes;
    static constexpr int kSfaBytes = 2 * kSfTile, kSfbBytes = 4 * kSfTile;
    static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
    static constexpr int kOutBytes = kEpiWarps * kChunk * 64;
    static constexpr int kVecBytes = kEpiWarps * kMaxChunks * 2 * kChunk * 4;
    static constexpr int kStages = 5, kSlots = 4;
    static constexpr int kSfCols = 24;
    static constexpr int kAcc1 = 512 - kSlots * kSfCols - kTN;  // 160
    static constexpr int kSfCol0 = kAcc1 + kTN;                 // 416
    static_assert(kTN - kAcc1 <= kGroups * kChunk, "the first chunks hold every shared column");
    static constexpr int kAOff = 0;
    static constexpr int kBOff = kAOff + kStages * kABytes;
    static constexpr int kOutOff = kBOff + kStages * kBBytes;
    static constexpr int kSfaOff = kOutOff + kOutBytes;
    static constexpr int kSfbOff = kSfaOff + kStages * kSfaBytes;
    static constexpr int kVecOff = kSfbOff + kStages * kSfbBytes;
    static constexpr int kBarOff = kVecOff + kVecBytes;
    static constexpr int kNumBars = 2 * kStages + 4 + 1 + 1 + kEpiWarps;
    static constexpr int kSmemBytes = kBarOff + kNumBars * 8 + 16 + 1024;
    static_assert(kSmemBytes <= 232448, "shared memory");
    static constexpr uint32_t kIdesc = idesc_mxf4(2 * kTM, kTN);
};

__device__ __forceinline__ void tc_copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void tc_mma_mxf4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                                 uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// 3-D tiled load by either CTA of a pair, completion counted on a barrier of either (no multicast).
__device__ __forceinline__ void tma_load_3d_pair(void *dst, const CUtensorMap *map, uint32_t bar_cluster, int32_t c0, int32_t c1, int32_t c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

template <bool TMA>
__global__ void __launch_bounds__(PairCfg::kThreads, 1)
    mx4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                         const __grid_constant__ CUtensorMap tmap_sfa, const __grid_constant__ CUtensorMap tmap_sfb,
                         const __grid_constant__ CUtensorMap tmap_y, const __grid_constant__ CUtensorMap tmap_res, const Params p) {
    using C = PairCfg;
    constexpr int S = C::kStages, TN = C::kTN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::kBarOff);  // [S] leader: both CTAs' stage landed
    uint64_t *empty = full + S;                                        // [S] stage's MMAs complete (both CTAs)
    uint64_t *acc_full = empty + S;                                    // [2] (both CTAs)
    uint64_t *acc_empty = acc_full + 2;                                // [2] leader: drained by both CTAs
    uint64_t *shared_cols = acc_empty + 2;                             // leader: a tile's shared columns are in registers
    uint64_t *drain = shared_cols + 1;
    uint64_t *res_full = drain + 1;                                    // [warp] residual chunk landed
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(res_full + C::kEpiWarps);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int unit = (int)cluster_id_x(), units = (int)cluster_count_x();

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * C::kEpiWarps);
        }
        mbar_init(shared_cols, 2 * C::kEpiWarps);
        mbar_init(drain, 1);
        for (int i = 0; i < C::kEpiWarps; ++i) mbar_init(&res_full[i], 1);
        fence_barrier_init();
    }
    if (warp == C::kMma) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    if (warp == C::kProducer && lane == 0) {
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
        tma_prefetch_desc(&tmap_sfa);
        tma_prefetch_desc(&tmap_sfb);
        if (TMA) tma_prefetch_desc(&tmap_y);
        if (TMA && p.ep.residual) tma_prefetch_desc(&tmap_res);
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();  // barriers initialised and tensor memory allocated in both CTAs
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const int tiles = p.m_tiles * p.n_tiles;

    if (warp == C::kProducer) {
        // ------------------------------------------------------------ producer
        pdl_dependency_wait();
        uint32_t i = 0;
        bool ok = true;
        for (int t = unit; ok && t < tiles; t += units) {
            int mt, nt;
            tile_at(p, t, mt, nt);
            const int m0 = mt * (2 * kTM) + (int)rank * kTM, n0 = nt * TN;
            for (int kb = 0; kb < p.nkb; ++kb, ++i) {
                const int s = i % S;
                if (!mbar_wait<true>(&empty[s], ((i / S) & 1) ^ 1, p.err, kErrTimeoutProducer)) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
                    if (leader) mbar_arrive_expect_tx(&full[s], 2 * C::kStageBytes);
                    tma_load_2d_pair(smem + C::kAOff + s * C::kABytes, &tmap_a, bar, kb * kRowBytes, m0);
                    tma_load_2d_pair(smem + C::kBOff + s * C::kBBytes, &tmap_b, bar, kb * kRowBytes, n0 + (int)rank * (TN / 2));
                    tma_load_3d_pair(smem + C::kSfaOff + s * C::kSfaBytes, &tmap_sfa, bar, 0, kb * 4, m0 >> 7);
                    tma_load_3d_pair(smem + C::kSfbOff + s * C::kSfbBytes, &tmap_sfb, bar, 0, kb * 4, n0 >> 7);
                }
                __syncwarp();
            }
        }
        pdl_launch_dependents();
        if (!ok && leader) {  // let the pair's copies already issued land before either CTA exits
            const uint32_t first = i > (uint32_t)S ? i - S : 0;
            for (uint32_t j = first; j < i; ++j) mbar_wait<true>(&full[j % S], (j / S) & 1, p.err, kErrTimeoutDrain);
        }
    } else if (warp == C::kMma) {
        // ------------------------------------------------------------ MMA issuer
        if (leader) {
            bool ok = true, issued = false;
            uint32_t i = 0;
            int lt = 0;
            constexpr uint16_t kBoth = 0x3;
            const uint64_t adesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kAOff)), bdesc0 = sdesc_kmajor_sw128(smem_u32(smem + C::kBOff));
            const uint64_t sadesc0 = sdesc_scales(smem_u32(smem + C::kSfaOff)), sbdesc0 = sdesc_scales(smem_u32(smem + C::kSfbOff));
            for (int t = unit; ok && t < tiles; t += units, ++lt) {
                const int b = lt & 1;
                ok = mbar_wait<true>(&acc_empty[b], ((lt >> 1) & 1) ^ 1, p.err, kErrTimeoutMma);
                if (ok && lt > 0) ok = mbar_wait<true>(shared_cols, (lt - 1) & 1, p.err, kErrTimeoutMma);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t d = tmem + (b ? C::kAcc1 : 0);
                uint32_t acc = 0;
                for (int kb = 0; kb < p.nkb; ++kb, ++i) {
                    const uint32_t s = i % S;
                    ok = mbar_wait<true>(&full[s], (i / S) & 1, p.err, kErrTimeoutMma);
                    // The slot's last MMAs, kSlots stages ago, are complete.
                    if (ok && i >= C::kSlots) ok = mbar_wait<true>(&empty[(i - C::kSlots) % S], ((i - C::kSlots) / S) & 1, p.err, kErrTimeoutMma);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after_sync();
                    if (lane_elect()) {
                        const uint32_t sfa = tmem + C::kSfCol0 + i % C::kSlots * C::kSfCols, sfb = sfa + 8;
                        const uint64_t ad = adesc0 + (uint64_t)s * (C::kABytes >> 4), bd = bdesc0 + (uint64_t)s * (C::kBBytes >> 4);
                        const uint64_t sad = sadesc0 + (uint64_t)s * (C::kSfaBytes >> 4), sbd = sbdesc0 + (uint64_t)s * (C::kSfbBytes >> 4);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {  // 128 columns: one scale tile along k
                            tc_copy_scales_pair(sfa + h * 4, sad + h * (kSfTile >> 4));
#pragma unroll
                            for (int j = 0; j < 2; ++j) tc_copy_scales_pair(sfb + h * 8 + j * 4, sbd + (j * 2 + h) * (kSfTile >> 4));
                        }
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const uint32_t id = idesc_scale_id((kk & 1) * 2);
                            tc_mma_mxf4_pair(d, ad + kk * 2, bd + kk * 2, C::kIdesc | id, sfa + (kk >> 1) * 4,
                                             sfb + (kk >> 1) * 8, acc);
                            acc = 1;
                        }
                        tc_commit_pair_multicast(&empty[s], kBoth);
                    }
                    acc = 1;
                    issued = true;
                }
                if (!ok) break;
                if (lane_elect()) tc_commit_pair_multicast(&acc_full[b], kBoth);
                __syncwarp();
            }
            if (!ok && issued) {
                if (lane_elect()) tc_commit_pair_multicast(drain, 0x1);
                __syncwarp();
                mbar_wait<true>(drain, 0, p.err, kErrTimeoutDrain);
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue
        pdl_dependency_wait();
        const int quad = warp & 3, group = warp >> 2;
        const ChunkOut o{smem + C::kOutOff + warp * kChunk * 64, reinterpret_cast<float *>(smem + C::kVecOff) + warp * C::kMaxChunks * 2 * kChunk,
                         res_full + warp};
        uint32_t q = 0;
        int lt = 0;
        for (int t = unit; t < tiles; t += units, ++lt) {
            int mt, nt;
            tile_at(p, t, mt, nt);
            const int m0 = mt * (2 * kTM) + (int)rank * kTM + quad * 32, n0 = nt * TN;
            const int b = lt & 1;
            // From the last chunk down in the first accumulator, from the first up in the second: the shared columns are
            // the first that are taken.
            auto place = [&](int c) {
                const int i = C::kGroups * c + group;
                return kChunk * (b ? i : TN / kChunk - 1 - i);
            };
            auto feature = [&](int c) { return C::kGroups * c + group < TN / kChunk ? n0 + place(c) : INT_MAX - kChunk; };
            auto column = [&](int c) { return ((uint32_t)(quad * 32) << 16) + (b ? C::kAcc1 : 0) + place(c); };
            auto loaded = [&](int c) {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0 && c != 1) mbar_arrive_cluster(mapa_shared(smem_u32(c == 0 ? shared_cols : &acc_empty[b]), 0));
            };
            if (!tile_epilogue<true, TMA, C::kMaxChunks>(p, &tmap_y, &tmap_res, o, &acc_full[b], (lt >> 1) & 1, tmem, m0, q, feature, column, loaded)) break;
        }
        if (lane == 0) bulk_wait_all();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();  // the peer's arrivals, copies and MMAs on this CTA are over
    if (warp == C::kMma) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem, 512);
    }
}

// Rows of y and the residual on 16-byte boundaries.
static bool by_tma(int64_t n) { return n % 8 == 0; }

// Scales as [row tiles][256-byte rows]: a stage's two tiles of a row tile are four consecutive rows.
static qmm_status map_scales(CUtensorMap *map, const uint8_t *scales, int64_t rows, int64_t k, uint32_t row_tiles_a_box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(QMM_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t per = (cuuint64_t)mx4_scale_tiles(k) * 2;
    cuuint64_t dims[3] = {256, per, (cuuint64_t)mx4_row_tiles(rows)};
    cuuint64_t strides[2] = {256, per * 256};
    cuuint32_t box[3] = {256, 4, row_tiles_a_box};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(scales), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(QMM_ERR_CUDA, "cuTensorMapEncodeTiled (scales) failed (%d)", (int)r);
    return QMM_OK;
}

// Tensor maps of the operands and output, and what both kernels need to know.
struct Problem {
    CUtensorMap a, b, y, res;
    Params p;
};

static qmm_status make_problem(Problem &q, const qmm_mx4 &w, const qmm_mx4 &x, const qmm_epilogue &ep, uint16_t *y, int tm, int tn, int b_rows) {
    const uint64_t pitch = (uint64_t)mx4_pitch(w.k);
    qmm_status s = map_2d(&q.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, x.codes, pitch, (uint64_t)x.rows, pitch, kRowBytes, kTM, CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != QMM_OK) return s;
    s = map_2d(&q.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, w.codes, pitch, (uint64_t)w.rows, pitch, kRowBytes, (uint32_t)b_rows, CU_TENSOR_MAP_SWIZZLE_128B);
    if (s != QMM_OK) return s;
    q.y = q.res = q.a;
    if (by_tma(w.rows)) {
        s = map_2d(&q.y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, y, (uint64_t)w.rows, (uint64_t)x.rows, (uint64_t)w.rows * 2, kChunk, 32, CU_TENSOR_MAP_SWIZZLE_64B);
        if (s == QMM_OK && ep.residual)
            s = map_2d(&q.res, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ep.residual, (uint64_t)w.rows, (uint64_t)x.rows, (uint64_t)w.rows * 2, kChunk, 32,
                       CU_TENSOR_MAP_SWIZZLE_64B);
        if (s != QMM_OK) return s;
    }
    Params &p = q.p;
    p.a_scales = x.scales;
    p.b_scales = w.scales;
    p.ep = epilogue_args(ep);
    p.y = y;
    p.m = (int32_t)x.rows;
    p.n = (int32_t)w.rows;
    p.nkb = (int32_t)((w.k + kBK - 1) / kBK);
    p.sf_tiles = (int32_t)mx4_scale_tiles(w.k);
    const int64_t mt = (x.rows + tm - 1) / tm, nt = (w.rows + tn - 1) / tn;
    if (mt * nt > INT32_MAX / 2) return fail(QMM_ERR_UNSUPPORTED, "mxfp4 linear: too many output tiles");
    p.m_tiles = (int32_t)mt;
    p.n_tiles = (int32_t)nt;
    p.b_row_tiles = (int32_t)mx4_row_tiles(w.rows);
    p.err = device_error_word();
    return QMM_OK;
}

template <int TN, bool TMA>
static qmm_status launch_gemm(const qmm_mx4 &w, const qmm_mx4 &x, const qmm_epilogue &ep, uint16_t *y, cudaStream_t st) {
    using C = Cfg<TN>;
    static bool configured[64] = {};
    qmm_status s = allow_smem(mx4_gemm_kernel<TN, TMA>, C::kSmemBytes, configured);
    if (s != QMM_OK) return s;
    Problem q;
    s = make_problem(q, w, x, ep, y, kTM, TN, TN);
    if (s != QMM_OK) return s;
    const unsigned grid = (unsigned)std::min<int64_t>((int64_t)q.p.m_tiles * q.p.n_tiles, sm_count());
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, mx4_gemm_kernel<TN, TMA>, q.a, q.b, q.y, q.res, q.p);
    count_launch();
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? QMM_OK : cuda_fail(e, "mxfp4 gemm launch");
}

template <bool TMA>
static qmm_status launch_gemm_pair(const qmm_mx4 &w, const qmm_mx4 &x, const qmm_epilogue &ep, uint16_t *y, cudaStream_t st) {
    using C = PairCfg;
    static bool configured[64] = {};
    qmm_status s = allow_smem(mx4_gemm_pair_kernel<TMA>, C::kSmemBytes, configured);
    if (s != QMM_OK) return s;
    Problem q;
    s = make_problem(q, w, x, ep, y, 2 * kTM, C::kTN, C::kTN / 2);
    if (s != QMM_OK) return s;
    CUtensorMap sfa, sfb;
    if ((s = map_scales(&sfa, x.scales, x.rows, x.k, 1)) != QMM_OK) return s;
    if ((s = map_scales(&sfb, w.scales, w.rows, w.k, 2)) != QMM_OK) return s;
    const unsigned pairs = (unsigned)std::min<int64_t>((int64_t)q.p.m_tiles * q.p.n_tiles, std::max(1, sm_count() / 2));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = dim3(pairs * 2, 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, mx4_gemm_pair_kernel<TMA>, q.a, q.b, sfa, sfb, q.y, q.res, q.p);
    count_launch();
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? QMM_OK : cuda_fail(e, "mxfp4 gemm launch");
}

// Whether pairs of CTAs take the product in less time: turns of tiles over the device,
// each as long as its products, 2.0 ns a column of k with either tile, or, where k is
// short, its epilogue: 4.3 us (7 with an activation) for a CTA of a pair, 1.7 (2.9) for
// 128 x 192.  B200, pairs against single CTAs, without and with an activation: 16384 x
// 1536 -> 12288 190 (249) us against 172 (180), x 3072 264 (281) against 306 (331); 2000 x
// 3000 -> 5000, three turns of either, 23.6 against 20.5.
static bool pairs_take(int64_t m, int64_t k, int64_t n, bool act) {
    auto turns = [](int64_t tiles, int64_t places) { return (tiles + places - 1) / places; };
    const int64_t pair = turns(((m + 255) / 256) * ((n + 255) / 256), std::max(1, sm_count() / 2));
    const int64_t single = turns(((m + kTM - 1) / kTM) * ((n + 191) / 192), sm_count());
    return pair * std::max<int64_t>(k, act ? 3500 : 2150) < single * std::max<int64_t>(k, act ? 1450 : 850);
}

static qmm_status launch_product(const qmm_mx4 &w, const qmm_mx4 &x, const qmm_epilogue &ep, uint16_t *y, cudaStream_t st) {
    if (mx4_small_fits(w.rows, x.rows)) return launch_mx4_small(w, nullptr, 0, 0, x, ep, y, st);
    const bool tma = by_tma(w.rows);
    if (pairs_take(x.rows, w.k, w.rows, ep.activation != QMM_ACT_NONE))
        return tma ? launch_gemm_pair<true>(w, x, ep, y, st) : launch_gemm_pair<false>(w, x, ep, y, st);
    return tma ? launch_gemm<192, true>(w, x, ep, y, st) : launch_gemm<192, false>(w, x, ep, y, st);
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

uint64_t qmm_mx4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    return qmm::mx4::mx4_small_fits(n, m) && qmm::mx4::mx4_small_quantises(n, m, k) ? 0 : qmm_mx4_workspace_bytes(m, k);
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
    const uint64_t need = quantised ? 0 : qmm_mx4_linear_workspace_bytes(a.m, a.w.rows, a.w.k);
    if (!quantised) sx[0] = span(a.x, ((uint64_t)(a.m - 1) * (uint64_t)a.x_row_stride + (uint64_t)a.w.k) * xsize);
    if (need) {
        if (!a.workspace || a.workspace_bytes < need)
            return fail(QMM_ERR_INVALID_ARGUMENT, "mxfp4 linear: workspace of %llu bytes is smaller than %llu", (unsigned long long)a.workspace_bytes, (unsigned long long)need);
        if (misaligned(a.workspace)) return fail(QMM_ERR_MISALIGNED, "mxfp4 linear: workspace is not 16-byte aligned");
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
    const qmm_epilogue ep{a.bias, a.gate, a.residual, a.activation};
    if (!quantised && !need) return qmm::mx4::launch_mx4_small(a.w, a.x, a.x_elem, a.x_row_stride, x, ep, a.y, st);
    if (need) {
        s = qmm::launch_mx4_quantize(a.x, a.x_elem, a.m, a.w.k, a.x_row_stride, const_cast<uint8_t *>(x.codes), const_cast<uint8_t *>(x.scales), st);
        if (s != QMM_OK) return s;
    }
    return qmm::mx4::launch_product(a.w, x, ep, a.y, st);
}

}  // extern "C"
