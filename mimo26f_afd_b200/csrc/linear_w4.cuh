// Dense products with MXFP4 weights: y = x W^T, and the gated pair silu(x Wg^T) * (x Wu^T).
//
//     y[t, n] = sum_k x[t, k] * E2M1(w[n, k]) * 2^(s[n, k / 32] - 127)
//
// BF16 activations without an activation quantiser. The block-scaled MMA takes the 4-bit weights and their scale bytes as
// they are, but its other operand has at most 8 bits, so a K32 block of x is written as TWO E4M3 pieces with UE8M0 scales,
//     x = 2^s (hi + 2^-4 lo),   hi = E4M3(x / 2^s),   lo = E4M3(16 (x / 2^s - hi)),
// s the smallest exponent with max|x| <= 448 * 2^s. A BF16 significand has 8 bits: hi takes the leading four, and what is
// left of the other four (a signed value of at most 8 units in the last BF16 place) fits E4M3 again. So the pair IS x for
// every element of at least 2^-6 * 2^s, that is 2^-14 of its block's largest; below, the pair is off by at most
// 2^-14 * 2^s < 2^-21 of that largest element, what one FP32 rounding of a partial sum costs. Both pieces accumulate into
// the same FP32 tensor-memory tile: the weights are fetched once and the tensor pipe runs them twice, at the FP8 rate, which is
// the rate of a BF16 product - with no dequantised copy of the weights anywhere. Quantised activations (E4M3 rows with
// UE8M0 K32 scales) take one piece.
//
// A K32 block with an infinity or a NaN becomes a block of NaN: every output of that row is NaN.
//
// Weights are the MMA "A" operand (M = 128 rows per tile), tokens the "B" operand (N = token tile), as in gemm_mx.cuh.
// For the gated form a 128-row tile holds 64 gate rows and the 64 up rows of the same features.
#pragma once
#include "gemm_mx.cuh"
#include "block_norm.cuh"

namespace m26b {

// ---- weight image ------------------------------------------------------------------------------------------------
// payload [m_pairs][256 rows][k_pad / 2]: rows of two consecutive 128-row tiles, or (gated) 128 gate rows, then the up rows of
// the same 128 features. Rows beyond n and columns beyond k are zero.
// scales  [m_pairs][chunks][2][512]; gated: [m_pairs][2 halves][chunks][512], rows 0..63 of a block gate, 64..127 up.
struct LinearSrc { const uint8_t *w[2], *s[2]; };    // gate / up, or one matrix

__global__ void __launch_bounds__(256) linear_prep_payload_kernel(LinearSrc src, int gated, uint32_t n, uint32_t k, uint32_t k_pad, uint64_t rows,
                                                                  uint8_t* __restrict__ dst) {
    const uint64_t vec_per_row = k_pad / 32, total = rows * vec_per_row;
    for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += uint64_t(gridDim.x) * blockDim.x) {
        const uint64_t v = i % vec_per_row, row = i / vec_per_row;
        const int m = gated ? int((row >> 7) & 1) : 0;
        const uint64_t feat = gated ? (row >> 8) * 128 + (row & 127) : row;
        uint32_t o[4] = {0, 0, 0, 0};
        if (feat < n && v * 32 < k) {
            const uint8_t* from = src.w[m] + feat * (k / 2) + v * 16;
#pragma unroll
            for (int b = 0; b < 16; ++b) o[b >> 2] |= uint32_t(from[b]) << (8 * (b & 3));   // the source may have any alignment
        }
        reinterpret_cast<uint4*>(dst)[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}
__global__ void __launch_bounds__(256) linear_prep_scales_kernel(LinearSrc src, int gated, uint32_t n, uint32_t k, uint32_t chunks, uint64_t total,
                                                                 uint8_t* __restrict__ dst) {
    for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += uint64_t(gridDim.x) * blockDim.x) {
        const uint32_t o = uint32_t(i % kScaleBlockBytes);
        const uint32_t r = (o >> 4) + 32u * ((o >> 2) & 3u), kb = o & 3u;
        uint64_t feat, c;
        int m = 0;
        if (gated) {
            c = (i / kScaleBlockBytes) % chunks;
            const uint64_t ph = i / kScaleBlockBytes / chunks;                 // pair * 2 + half
            feat = (ph >> 1) * 128 + (ph & 1) * 64 + (r & 63u);
            m = int(r >> 6);
        } else {
            c = (i / kScaleBlockBytes / 2) % chunks;
            feat = (i / kScaleBlockBytes / 2 / chunks) * 256 + ((i / kScaleBlockBytes) & 1) * 128 + r;
        }
        const uint64_t kb_all = c * 4 + kb;
        uint8_t v = 127;
        if (feat < n && kb_all * 32 < k) v = src.s[m][feat * (k / 32) + kb_all];
        dst[i] = v == 255 ? 254 : v;                                           // the reserved byte, as in the layer image
    }
}

// ---- activations -> E4M3 pieces ------------------------------------------------------------------------------------
// Scale byte of the leading piece for a block maximum (bits of a finite FP32 magnitude); the second piece's byte is 4 less.
__device__ __forceinline__ uint32_t split_scale_byte(uint32_t amax_bits) {
    if (!amax_bits) return 127u;
    uint32_t sig; int exp;
    split_f32(amax_bits, sig, exp);
    const int s = exp - ((sig & 0x7fffffu) <= 0x600000u ? 8 : 7) + 127;
    return uint32_t(s < 4 ? 4 : s);                                            // at most 247
}
__device__ __forceinline__ uint32_t e4m3x2_rn(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_f32(uint32_t pair) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(pair)));
    float lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
    return make_float2(lo, hi);
}
// Eight BF16 values (bits in the upper half of FP32 words) with the block's scale byte -> eight codes of each piece.
__device__ __forceinline__ void split8(const float (&v)[8], uint32_t scale, bool bad, uint2& hi, uint2& lo) {
    if (bad) { hi = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu); lo = make_uint2(0, 0); return; }
    const float inv = __uint_as_float((254u - scale) << 23);                   // 2^(127 - scale), scale in 4..247
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = v[2 * j] * inv, b = v[2 * j + 1] * inv;
        h[j] = e4m3x2_rn(a, b);
        const float2 d = e4m3x2_f32(h[j]);
        l[j] = e4m3x2_rn((a - d.x) * 16.0f, (b - d.y) * 16.0f);
    }
    hi = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    lo = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
}

struct SplitArgs {
    const void* x;
    const uint8_t* x_scales;     // PIECES 1: [rows][k / 32]
    uint64_t pitch;              // elements
    int vec;                     // rows start on 16-byte (BF16) / 8-byte (E4M3) boundaries
    uint32_t rows, k, k_pad, rows_cap;
    uint8_t* q;                  // [PIECES][rows_cap][k_pad]
    uint8_t* sf;                 // [128-token tile][chunk][PIECES][512]
};
// Four threads per K32 block, eight elements each.
template <int PIECES>
__global__ void __launch_bounds__(256) linear_split_kernel(const SplitArgs p) {
    grid_dep_launch();
    const uint32_t groups = p.k_pad / 8;
    const uint64_t id = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    const uint64_t total = uint64_t(p.rows) * groups;      // a multiple of 16: the four threads of a block stay together
    if (id >= total) return;
    const uint32_t row = uint32_t(id / groups), g = uint32_t(id % groups), kb = g >> 2;
    const uint64_t at = uint64_t(row) * p.pitch + uint64_t(g) * 8;
    const bool real = g * 8 < p.k;
    uint32_t scale = 127;
    uint2 hi = make_uint2(0, 0), lo = make_uint2(0, 0);
    if constexpr (PIECES == 2) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        if (real) {
            if (p.vec) {
                load_elems<8>(p.x, 0, at, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(uint32_t(static_cast<const uint16_t*>(p.x)[at + e]) << 16);
            }
        }
        uint32_t amax = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(v[e]) & 0x7fffffffu);
        const uint32_t quad = 0xfu << (threadIdx.x & 28u);
        amax = max(amax, __shfl_xor_sync(quad, amax, 1));
        amax = max(amax, __shfl_xor_sync(quad, amax, 2));
        const bool bad = amax >= 0x7f800000u;
        if (!bad) scale = split_scale_byte(amax);
        split8(v, scale, bad, hi, lo);
    } else if (real) {
        const uint8_t* x = static_cast<const uint8_t*>(p.x) + at;
        if (p.vec) {
            hi = *reinterpret_cast<const uint2*>(x);
        } else {
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e >> 2] |= uint32_t(x[e]) << (8 * (e & 3));
            hi = make_uint2(o[0], o[1]);
        }
        scale = p.x_scales[uint64_t(row) * (p.k / 32) + kb];
        if (scale == 255u) { scale = 127; hi = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu); }      // a NaN scale
    }
    uint8_t* q = p.q + uint64_t(row) * p.k_pad + uint64_t(g) * 8;
    *reinterpret_cast<uint2*>(q) = hi;
    if constexpr (PIECES == 2) *reinterpret_cast<uint2*>(q + uint64_t(p.rows_cap) * p.k_pad) = lo;
    if ((g & 3u) == 0) {
        uint8_t* sf = p.sf + (uint64_t(row >> 7) * (p.k_pad / kChunkK) + (kb >> 2)) * PIECES * kScaleBlockBytes + scale_block_offset(int(row & 127u), int(kb & 3u));
        sf[0] = uint8_t(scale);
        if constexpr (PIECES == 2) sf[kScaleBlockBytes] = uint8_t(scale - 4u);
    }
}

// ---- the product ---------------------------------------------------------------------------------------------------
struct LinearArgs {
    const uint8_t* sfa;          // weight scales
    const uint8_t* sfb;          // token scales
    uint32_t rows, rows_cap;     // tokens of the pass; row offset of the second piece in the staged activations
    uint32_t n;                  // output width
    uint32_t chunks;             // k_pad / 128
    void* y;
    int y_f32;
    uint64_t y_pitch;            // elements
    uint32_t* fault;
};

__device__ __forceinline__ float silu_gate(float g, float u) {
    // g / (1 + e^-g) * u without a positive exponential; infinities of g give +inf * u and -0 * u
    const float e = __expf(-fabsf(g));
    const float s = __fdividef(g >= 0.0f ? 1.0f : e, 1.0f + e);
    return g * s * u;
}
__device__ __forceinline__ void store_y(const LinearArgs& p, uint32_t token, uint32_t col, float v) {
    const uint64_t at = uint64_t(token) * p.y_pitch + col;
    if (p.y_f32) static_cast<float*>(p.y)[at] = v;
    else static_cast<uint16_t*>(p.y)[at] = uint16_t(bf16x2_rn(v, 0.0f));
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <int B_ROWS, int PIECES>
struct LinearTile {
    static constexpr int kStageBytes = kTileM * 128 + PIECES * B_ROWS * 128 + (1 + PIECES) * kScaleBlockBytes;
    static constexpr int kCtasPerSm = B_ROWS <= 32 ? 2 : 1;
    static constexpr int kRedBytes = B_ROWS * kTileM * 4;          // partial sums of a split K, and the gate / up exchange
    static constexpr int kBudget = (kCtasPerSm == 2 ? 113 : 226) * 1024 - 2048;
    static constexpr int kFit = (kBudget - kRedBytes) / kStageBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr uint32_t kCols = B_ROWS + 32 <= 64 ? 64 : B_ROWS + 32 <= 128 ? 128 : 256;
    static_assert(kStages >= 3, "too few stages");
};
template <int B_ROWS, int PIECES>
struct LinearSmem {
    using T = LinearTile<B_ROWS, PIECES>;
    alignas(1024) uint8_t a[T::kStages][kTileM * 128];
    alignas(1024) uint8_t b[T::kStages][PIECES * B_ROWS * 128];
    alignas(128) uint8_t sfa[T::kStages][kScaleBlockBytes];
    alignas(128) uint8_t sfb[T::kStages][PIECES * kScaleBlockBytes];
    alignas(16) float red[T::kRedBytes / 4];
    uint64_t full[T::kStages], empty[T::kStages], acc_full;
    uint32_t tmem_base, abort_flag;
};
constexpr int kLinearThreads = 192;              // producer warp, MMA warp, four epilogue warps

// One CTA: one 128-row weight tile (blockIdx.x / split) x one token tile (blockIdx.y), over its share of the K chunks. The
// `split` CTAs of a cluster share a tile; they add their partial sums over distributed shared memory in rank order, CTA r
// finishing 1 / split of the tile's features, so the result does not depend on timing. Token tiles start on multiples of 128
// (their scale blocks hold 128 tokens): smaller B_ROWS serve requests of at most B_ROWS tokens.
template <int B_ROWS, int PIECES, bool GATED>
__global__ void __launch_bounds__(kLinearThreads, (LinearTile<B_ROWS, PIECES>::kCtasPerSm))
linear_w4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TokenMaps maps_x, const LinearArgs p, const uint32_t split) {
    using T = LinearTile<B_ROWS, PIECES>;
    using Smem = LinearSmem<B_ROWS, PIECES>;
    extern __shared__ uint8_t smem_raw[];
    Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = split > 1 ? cluster_ctarank() : 0;
    const uint32_t tile = blockIdx.x / split;
    const uint32_t c0 = p.chunks * rank / split, c1 = p.chunks * (rank + 1) / split;
    const uint32_t tok0 = blockIdx.y * B_ROWS;
    const uint32_t n_valid = p.rows - tok0 < B_ROWS ? p.rows - tok0 : B_ROWS, n_mma = (n_valid + 15) & ~15u;
    volatile uint32_t* abort_flag = &s.abort_flag;

    if (threadIdx.x == 0) {
        for (int i = 0; i < T::kStages; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
        mbar_init(&s.acc_full, 1);
        s.abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) { tmem_alloc(&s.tmem_base, T::kCols); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tb = s.tmem_base;
    if (split > 1) cluster_arrive();         // "this CTA has started": its shared memory may be written from now on

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (elect_one()) {
            tma_prefetch_desc(&map_w);
            const uint32_t n_chunks = c1 - c0;
            const uint32_t tx = kTileM * 64 + PIECES * n_mma * 128 + (1 + PIECES) * kScaleBlockBytes;
            const uint8_t* sfb_g = p.sfb + uint64_t(tok0 >> 7) * p.chunks * PIECES * kScaleBlockBytes;
            auto weights = [&](uint32_t i, uint32_t st) {
                const uint32_t c = c0 + i;
                mbar_expect_tx(&s.full[st], tx);
                if constexpr (GATED) {          // 64 gate rows, then the 64 up rows of the same features
                    tma_load_3d(s.a[st], &map_w, int(c * kChunkK), int((tile & 1) * 64), int(tile >> 1) * 2, &s.full[st]);
                    bulk_load(s.sfa[st], p.sfa + (uint64_t(tile) * p.chunks + c) * kScaleBlockBytes, kScaleBlockBytes, &s.full[st]);
                } else {
                    tma_load_2d(s.a[st], &map_w, int(c * kChunkK), int(tile * kTileM), &s.full[st]);
                    bulk_load(s.sfa[st], p.sfa + ((uint64_t(tile >> 1) * p.chunks + c) * 2 + (tile & 1)) * kScaleBlockBytes, kScaleBlockBytes, &s.full[st]);
                }
            };
            // the weights do not depend on the kernel that stages the activations: their first stages are requested before it ends
            const uint32_t early = n_chunks < uint32_t(T::kStages) ? n_chunks : uint32_t(T::kStages);
            for (uint32_t i = 0; i < early; ++i) weights(i, i);
            grid_dep_wait();
            uint32_t stage = 0, phase = 0;
            for (uint32_t i = 0; i < n_chunks; ++i) {
                if (i >= early) {
                    if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort_flag)) { atomicOr(p.fault, uint32_t(kFaultPipeline)); break; }
                    weights(i, stage);
                }
                const uint32_t c = c0 + i;
#pragma unroll
                for (int piece = 0; piece < PIECES; ++piece) {
                    uint32_t r = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const uint32_t box = 128u >> b;
                        if (box <= B_ROWS && n_mma - r >= box) {
                            tma_load_2d(s.b[stage] + (piece * B_ROWS + r) * 128, &maps_x.box[b], int(c * kChunkK),
                                        int(piece * p.rows_cap + tok0 + r), &s.full[stage]);
                            r += box;
                        }
                    }
                }
                bulk_load(s.sfb[stage], sfb_g + uint64_t(c) * PIECES * kScaleBlockBytes, PIECES * kScaleBlockBytes, &s.full[stage]);
                if (++stage == uint32_t(T::kStages)) { stage = 0; phase ^= 1u; }
            }
            if (*abort_flag) {                     // a wait ran out: leave no copy of this CTA in flight behind
                for (uint32_t i = 0; i < early; ++i) {
                    const long long t0 = clock64();
                    while (!mbar_try_wait(&s.full[i], 0) && clock64() - t0 < kWaitCycles) {}
                }
            }
        }
        __syncwarp();
        if (split > 1) cluster_wait();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issue
        if (elect_one()) {
            const uint32_t idesc0 = idesc_mx(kFmtE2M1, kFmtE4M3, n_mma, 0, 0);
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t c = c0; c < c1; ++c) {
                if (!mbar_wait(&s.full[stage], phase, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t t_sf = tb + B_ROWS + (c & 1u) * 16u;      // consecutive chunks alternate between two scale slots
                tc_cp_scales(t_sf, desc_scale_block(smem_u32(s.sfa[stage])));
#pragma unroll
                for (int piece = 0; piece < PIECES; ++piece) tc_cp_scales(t_sf + 4 + 4 * piece, desc_scale_block(smem_u32(s.sfb[stage]) + piece * kScaleBlockBytes));
                const uint64_t ad = desc_sw128(smem_u32(s.a[stage]));
#pragma unroll
                for (int piece = 0; piece < PIECES; ++piece) {
                    const uint64_t bd = desc_sw128(smem_u32(s.b[stage]) + piece * B_ROWS * 128);
#pragma unroll
                    for (uint32_t kb = 0; kb < 4; ++kb)
                        tc_mma_mx(tb, ad + 2 * kb, bd + 2 * kb, idesc0 | (kb << 4) | (kb << 29), t_sf, t_sf + 4 + 4 * piece, (c != c0 || piece || kb) ? 1u : 0u);
                }
                tc_commit(&s.empty[stage]);
                if (++stage == uint32_t(T::kStages)) { stage = 0; phase ^= 1u; }
            }
            if (ok) tc_commit(&s.acc_full);
            else atomicOr(p.fault, uint32_t(kFaultPipeline));
        }
        __syncwarp();
        if (split > 1) cluster_wait();
    } else {
        // ------------------------------------------------------------ epilogue, first half: tensor memory -> where it is added
        const uint32_t q = uint32_t(warp) & 3u;
        const uint32_t row = q * 32u + lane;               // weight row of the tile
        const bool ok = mbar_wait(&s.acc_full, 0, abort_flag);
        __syncwarp();
        if (split > 1) cluster_wait();
        if (__all_sync(0xffffffffu, ok)) {
            tc_fence_after();
            const uint32_t t_acc = tb + ((q * 32u) << 16);
            // owner of a row and its place there: features are dealt in equal runs, gate and up of a feature together
            const uint32_t per = kTileM / split;
            uint32_t owner, slot;
            if constexpr (GATED) {
                const uint32_t f = row & 63u, half = per / 2;
                owner = f / half; slot = (row >> 6) * half + f % half;
            } else {
                owner = row / per; slot = row % per;
            }
            const uint32_t base = split > 1 ? cluster_map(smem_u32(s.red), owner) : smem_u32(s.red);
            const uint32_t feat = tile * kTileM + row;
            for (uint32_t col = 0; col < n_mma; col += 16) {
                uint32_t r[16];
                tmem_ld16(t_acc + col, r);
                tmem_wait_ld();
                if (!GATED && split == 1) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (col + j < n_valid && feat < p.n) store_y(p, tok0 + col + j, feat, __uint_as_float(r[j]));
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        st_cluster_f32(base + ((rank * n_mma + col + j) * per + slot) * 4, __uint_as_float(r[j]));
                }
            }
            tc_fence_before();
        }
    }
    __syncthreads();
    if (warp == 1) tmem_dealloc(tb, T::kCols);
    if (!GATED && split == 1) return;
    if (split > 1) cluster_sync_all();
    // ------------------------------------------------------------ epilogue, second half: partial sums in rank order
    const uint32_t per = kTileM / split, feats = GATED ? per / 2 : per;
    const uint32_t feat0 = GATED ? tile * 64 + rank * feats : tile * kTileM + rank * feats;
    for (uint32_t i = threadIdx.x; i < n_valid * feats; i += kLinearThreads) {
        const uint32_t col = i / feats, f = i % feats;
        if (feat0 + f >= p.n) continue;
        float v = 0.0f, u = 0.0f;
        for (uint32_t r = 0; r < split; ++r) {
            const float* from = s.red + (r * n_mma + col) * per + f;
            v += from[0];
            if constexpr (GATED) u += from[feats];
        }
        store_y(p, tok0 + col, feat0 + f, GATED ? silu_gate(v, u) : v);
    }
}

}  // namespace m26b
