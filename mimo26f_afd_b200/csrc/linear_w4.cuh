// Dense products with MXFP4 weights: y = x W^T, and the gated pair silu(x Wg^T) * (x Wu^T).
//
//     y[t, n] = sum_k x[t, k] * E2M1(w[n, k]) * 2^(s[n, k / 32] - 127)
//
// BF16 activations without an activation quantiser. The block-scaled MMA takes the 4-bit weights and their scale bytes as
// they are, but its other operand has at most 8 bits, so a K32 block of x is written as TWO E4M3 pieces with UE8M0 scales,
//     x = 2^s (hi + 2^-4 lo),   hi = E4M3(x / 2^s),   lo = E4M3(16 (x / 2^s - hi)),
// s the smallest exponent with max|x| <= 448 * 2^s. A BF16 significand has 8 bits: hi takes the leading four, and what is
// left of the other four (a signed value of at most 8 units in the last BF16 place) fits E4M3 again. So the pair IS x for
// every element of at least 2^-6 * 2^s, so of at least 2^-13 of its block's largest; below, the pair is off by at most
// 2^-14 * 2^s < 2^-21 of that largest element, what one FP32 rounding of a partial sum costs. The products of both pieces
// accumulate in FP32 tensor memory: the weights are fetched once and the tensor pipe runs them twice, at the FP8 rate, which is
// the rate of a BF16 product - with no dequantised copy of the weights anywhere. Each piece has accumulators of its own. Quantised
// activations (E4M3 rows with UE8M0 K32 scales) take one piece.
//
// A K32 block with an infinity or a NaN becomes a block of NaN: every output of that row is NaN.
//
// Weights are the MMA "A" operand (M = 128 rows per tile), tokens the "B" operand (N = token tile), as in gemm_mx.cuh.
#pragma once
#include "gemm_mx.cuh"
#include "block_norm.cuh"

namespace m26b {

// ---- weight image ------------------------------------------------------------------------------------------------
// payload [tiles][128 rows][k_pad / 2], scales [tiles][chunks][512]. A tile is 128 consecutive output features; for the gated form
// it is 64 features, sixteen gate rows and then the sixteen up rows of the same features in every 32 (the lanes one warp reads
// from tensor memory), so that a feature's gate and up meet by one shuffle. Rows beyond n and columns beyond k are zero; the
// number of tiles is even.
struct LinearSrc { const uint8_t *w[2], *s[2]; };    // gate / up, or one matrix

// Which matrix and which of its features image row `row` holds.
__device__ __forceinline__ void image_row(uint64_t row, int gated, int& matrix, uint64_t& feat) {
    matrix = gated ? int((row >> 4) & 1) : 0;
    feat = gated ? (row >> 5) * 16 + (row & 15) : row;
}
__global__ void __launch_bounds__(256) linear_prep_payload_kernel(LinearSrc src, int gated, uint32_t n, uint32_t k, uint32_t k_pad, uint64_t rows,
                                                                  uint8_t* __restrict__ dst) {
    const uint64_t vec_per_row = k_pad / 32, total = rows * vec_per_row;
    for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += uint64_t(gridDim.x) * blockDim.x) {
        const uint64_t v = i % vec_per_row;
        int m;
        uint64_t feat;
        image_row(i / vec_per_row, gated, m, feat);
        uint32_t o[4] = {0, 0, 0, 0};
        if (feat < n && v * 32 < k) {
            const uint8_t* from = (m ? src.w[1] : src.w[0]) + feat * (k / 2) + v * 16;
            if ((reinterpret_cast<uintptr_t>(from) & 15) == 0) {
                const uint4 a = *reinterpret_cast<const uint4*>(from);
                o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
            } else {
#pragma unroll
                for (int b = 0; b < 16; ++b) o[b >> 2] |= uint32_t(from[b]) << (8 * (b & 3));
            }
        }
        reinterpret_cast<uint4*>(dst)[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}
__global__ void __launch_bounds__(256) linear_prep_scales_kernel(LinearSrc src, int gated, uint32_t n, uint32_t k, uint32_t chunks, uint64_t total,
                                                                 uint8_t* __restrict__ dst) {
    for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += uint64_t(gridDim.x) * blockDim.x) {
        const uint32_t o = uint32_t(i % kScaleBlockBytes);
        const uint64_t c = (i / kScaleBlockBytes) % chunks, kb = c * 4 + (o & 3u);
        int m;
        uint64_t feat;
        image_row(i / kScaleBlockBytes / chunks * kTileM + (o >> 4) + 32u * ((o >> 2) & 3u), gated, m, feat);
        uint8_t v = 127;
        if (feat < n && kb * 32 < k) v = (m ? src.s[1] : src.s[0])[feat * (k / 32) + kb];
        dst[i] = v == 255 ? 254 : v;                                           // the reserved byte, as in the layer image
    }
}

// ---- activations -> E4M3 pieces ------------------------------------------------------------------------------------
// Scale byte of the leading piece for a block maximum (bits of a finite FP32 magnitude); the second piece's byte is 4 less.
__device__ __forceinline__ uint32_t split_scale_byte(uint32_t amax_bits) {
    // exponent field - 8, one more when the significand is above 1.75 (448 = 1.75 * 2^8); zero and subnormal blocks end at the floor
    const int s = int((amax_bits + 0x1fffffu) >> 23) - 8;
    return uint32_t(s < 4 ? 4 : s);                                            // at most 247
}
__device__ __forceinline__ uint32_t e4m3x2_rn(uint32_t f16x2) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(f16x2));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint32_t pair) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(pair)));
    return h;
}
// Largest magnitude of a K32 block, as FP32 bits: each of the block's four neighbouring lanes holds eight BF16 (`lanes`: those four
// or more). Infinities and NaN order above every number.
__device__ __forceinline__ uint32_t block_amax(const uint32_t (&w)[4], uint32_t lanes) {
    uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    m = __vmaxu2(m, __shfl_xor_sync(lanes, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(lanes, m, 2));
    return max(m << 16, m & 0xffff0000u);
}
// Eight BF16 (pairs as in memory) under the block's scale byte -> eight codes of each piece. The scaled values, at most 448 with
// eight significant bits, are exact in FP16 down to 2^-17 and off by 2^-25 at most below, far under the second piece's 2^-13
// grid; their difference to the first piece is exact there too.
__device__ __forceinline__ void split8(const uint32_t (&w)[4], uint32_t scale, bool bad, uint2& hi, uint2& lo) {
    // 2^(127 - scale), scale in 4..247; a bad block is scaled by NaN and becomes NaN codes
    const float inv = bad ? __int_as_float(0x7fc00000) : __uint_as_float((254u - scale) << 23);
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t a, r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(a) : "f"(__uint_as_float(w[j] & 0xffff0000u) * inv), "f"(__uint_as_float(w[j] << 16) * inv));
        h[j] = e4m3x2_rn(a);
        asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(f16x2_of_e4m3x2(h[j])));
        asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0x4c004c00u));         // 16
        l[j] = e4m3x2_rn(r);
    }
    hi = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    lo = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
}

struct SplitArgs {
    const void* x;
    const uint8_t* x_scales;     // PIECES 1: [rows][k / 32]
    uint64_t pitch;              // elements
    uint32_t rows, k, k_pad, rows_cap;
    // Scale blocks: [token tile of `tile` tokens][chunk][128-token run of the tile][piece][512]; with `joint` (tiles of 64) one block holds both
    // pieces, the second's tokens from row 64 on.
    uint32_t tile, joint;
    uint8_t* q;                  // [PIECES][rows_cap][k_pad]
    uint8_t* sf;
};
// A warp takes one 128-wide chunk of eight rows: sixteen lanes per row, eight elements each, two rows at a time; all its loads are
// issued first. VEC: rows start on 16-byte (BF16) / 8-byte (E4M3) boundaries. What bounds it is HBM and L2: 8,192 x 4,096 BF16 reads 67 MB and
// writes 67 MB of codes in 26 us = 5.0 TB/s (a thread per eight elements, with the row and the tile found by division: 34 us).
template <int PIECES, bool VEC>
__global__ void __launch_bounds__(256) linear_split_kernel(const SplitArgs p) {
    grid_dep_wait();             // x, and the workspace that an earlier call may still read
    grid_dep_launch();
    const uint32_t lane = threadIdx.x & 31u, chunks = p.k_pad / kChunkK, c = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (c >= chunks) return;
    const uint32_t g = lane & 15u, col = c * kChunkK + g * 8, row0 = blockIdx.y * 8;
    const bool inside = col < p.k;
    const uint32_t t = row0 / p.tile, r0 = row0 - t * p.tile;                  // eight rows never straddle a tile: tiles are multiples of 16
    uint32_t w[4][PIECES == 2 ? 4 : 2], scale[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        uint32_t row = row0 + 2 * v + (lane >> 4);
        row = row < p.rows ? row : p.rows - 1;                                 // beyond the request: read its last row, write nothing
        const uint64_t at = uint64_t(row) * p.pitch + (inside ? col : 0);
        if constexpr (PIECES == 2) {
            const uint16_t* x = static_cast<const uint16_t*>(p.x) + at;
            if constexpr (VEC) {
                const uint4 a = *reinterpret_cast<const uint4*>(x);
                w[v][0] = a.x; w[v][1] = a.y; w[v][2] = a.z; w[v][3] = a.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[v][e] = uint32_t(x[2 * e]) | uint32_t(x[2 * e + 1]) << 16;
            }
            scale[v] = 127;
        } else {
            const uint8_t* x = static_cast<const uint8_t*>(p.x) + at;
            if constexpr (VEC) {
                const uint2 a = *reinterpret_cast<const uint2*>(x);
                w[v][0] = a.x; w[v][1] = a.y;
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) w[v][e] = uint32_t(x[4 * e]) | uint32_t(x[4 * e + 1]) << 8 | uint32_t(x[4 * e + 2]) << 16 | uint32_t(x[4 * e + 3]) << 24;
            }
            scale[v] = p.x_scales[uint64_t(row) * (p.k / kBlockK) + (inside ? col : 0) / kBlockK];
        }
    }
    uint2 hi[4], lo[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
#pragma unroll
        for (uint32_t& word : w[v]) word = inside ? word : 0u;
        if constexpr (PIECES == 2) {
            const uint32_t amax = block_amax(w[v], 0xffffffffu);
            const bool bad = amax >= 0x7f800000u;
            scale[v] = bad ? 127u : split_scale_byte(amax);
            split8(w[v], scale[v], bad, hi[v], lo[v]);
        } else {
            const bool nan = inside && scale[v] == 255u;                       // a NaN scale
            scale[v] = nan || !inside ? 127u : scale[v];
            hi[v] = nan ? make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu) : make_uint2(w[v][0], w[v][1]);
        }
    }
    uint8_t* sf = p.sf + (uint64_t(t) * chunks + c) * (p.joint ? 1 : (p.tile + 127) / 128 * PIECES) * kScaleBlockBytes + (r0 >> 7) * PIECES * kScaleBlockBytes;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const uint32_t own = lane & 16u, row = row0 + 2 * v + (own >> 4), r = (r0 & 127u) + 2 * v + (own >> 4);
        uint32_t word = 0;                                                     // the row's four scale bytes of the chunk
#pragma unroll
        for (int b = 0; b < 4; ++b) word |= __shfl_sync(0xffffffffu, scale[v], own + 4 * b) << (8 * b);
        if (row >= p.rows) continue;
        uint8_t* q = p.q + uint64_t(row) * p.k_pad + col;
        *reinterpret_cast<uint2*>(q) = hi[v];
        if constexpr (PIECES == 2) *reinterpret_cast<uint2*>(q + uint64_t(p.rows_cap) * p.k_pad) = lo[v];
        if (g == 0) {
            *reinterpret_cast<uint32_t*>(sf + scale_block_offset(int(r), 0)) = word;
            if constexpr (PIECES == 2) {                                       // every byte is at least 4
                uint8_t* sl = p.joint ? sf + scale_block_offset(int(64 + r), 0) : sf + kScaleBlockBytes + scale_block_offset(int(r), 0);
                *reinterpret_cast<uint32_t*>(sl) = word - 0x04040404u;
            }
        }
    }
}

// Quantised activations whose rows TMA can take where they are (16-byte boundaries): only their scale bytes are staged, one thread per
// row and chunk. Byte 255 is a NaN to the MMA too.
__global__ void __launch_bounds__(256) linear_scales_kernel(const SplitArgs p) {
    grid_dep_wait();             // the scales, and the workspace that an earlier call may still read
    grid_dep_launch();
    const uint32_t chunks = p.k_pad / kChunkK, blocks = p.k / kBlockK, row = blockIdx.y * 8 + (threadIdx.x >> 5), c = blockIdx.x * 32 + (threadIdx.x & 31u);
    if (row >= p.rows || c >= chunks) return;
    const uint8_t* from = p.x_scales + uint64_t(row) * blocks;
    uint32_t word = 0;
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) word |= (4 * c + b < blocks ? uint32_t(from[4 * c + b]) : 127u) << (8 * b);
    const uint32_t t = row / p.tile, r = row - t * p.tile;
    uint8_t* sf = p.sf + ((uint64_t(t) * chunks + c) * ((p.tile + 127) / 128) + (r >> 7)) * kScaleBlockBytes;
    *reinterpret_cast<uint32_t*>(sf + scale_block_offset(int(r & 127u), 0)) = word;
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
    // activations as the caller has them (DIRECT kernels): rows start on 16-byte (BF16) / 8-byte (E4M3) boundaries
    const void* x;
    const uint8_t* x_scales;
    uint64_t x_pitch;
    uint32_t k;
    long long wait_cycles;       // bound of the epilogue's wait for its accumulators
};

// An epilogue warp's wait for finished accumulators. If it takes longer than p.wait_cycles, or another role has given up, that is
// reported and the answer is false; what is under way is waited for all the same (with the common bound), so that nothing
// of the tensor core or the copies is in flight when the kernel ends.
__device__ __forceinline__ bool acc_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, const LinearArgs& p) {
    const long long t0 = clock64();
    bool done, in_time;
    do {
        done = mbar_try_wait(bar, parity);
        in_time = clock64() - t0 <= p.wait_cycles;
    } while (!done && in_time && !*abort_flag);
    if (done && in_time) return true;
    atomicOr(p.fault, uint32_t(kFaultPipeline));
    if (!done) mbar_wait(bar, parity, abort_flag);
    return false;
}

// g / (1 + e^-g) * u without a positive exponential, within 2^-19 of itself for every g. expf and not the approximation, whose error grows
// with |g| (2^-18 at -60). `near`: g >= -64, where e^g is a normal number; an infinite g gives inf * u. `far`: any g; e^(g / 2) is met
// twice, so that g e^g u is whole where e^g alone has left FP32. Below -512 nothing is left whatever u is: -inf gives -0 * u.
constexpr float kSiluFar = -64.0f;
__device__ __forceinline__ float silu_near(float g, float u) {
    const float e = expf(-fabsf(g));
    return g * __fdividef(g >= 0.0f ? 1.0f : e, 1.0f + e) * u;
}
__device__ __forceinline__ float silu_far(float g, float u) {
    const float c = g < -512.0f ? -512.0f : g, h = expf(-0.5f * fabsf(c)), d = c >= 0.0f ? 1.0f : h;
    return __fdividef(c * d, fmaf(h, h, 1.0f)) * u * d;
}
__device__ __forceinline__ float silu_gate(float g, float u) { return g < kSiluFar ? silu_far(g, u) : silu_near(g, u); }
__device__ __forceinline__ void store_y(const LinearArgs& p, uint32_t token, uint32_t col, float v) {
    const uint64_t at = uint64_t(token) * p.y_pitch + col;
    if (p.y_f32) static_cast<float*>(p.y)[at] = v;
    else static_cast<uint16_t*>(p.y)[at] = uint16_t(bf16x2_rn(v, 0.0f));
}
// Sixteen finished accumulator columns (tokens from `token`, valid below `end`) of the lane's weight row. Gated: lanes 0..15 hold the
// gate of sixteen features and lanes 16..31 their up; of every two tokens the lower half finishes the first, the upper the second.
template <bool GATED>
__device__ __forceinline__ void store_columns(const LinearArgs& p, const uint32_t (&r)[16], uint32_t token, uint32_t end, uint32_t feat, int lane) {
    if constexpr (GATED) {
        const bool upper = lane >= 16;
        float g[8], u[8], low = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float other = __uint_as_float(__shfl_xor_sync(0xffffffffu, upper ? r[2 * j] : r[2 * j + 1], 16));
            const float mine = __uint_as_float(upper ? r[2 * j + 1] : r[2 * j]);
            g[j] = upper ? other : mine;
            u[j] = upper ? mine : other;
            low = fminf(low, g[j]);
        }
        if (__builtin_expect(low < kSiluFar, 0)) {       // asked once for the eight: hardly any gate is
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = silu_gate(g[j], u[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = silu_near(g[j], u[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t t = token + 2 * j + (upper ? 1 : 0);
            if (t < end && feat < p.n) store_y(p, t, feat, u[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (token + j < end && feat < p.n) store_y(p, token + j, feat, __uint_as_float(r[j]));
    }
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// The pieces of a token tile are one MMA operand of PIECES * B_ROWS rows - the second piece's B_ROWS rows behind the first's - with
// accumulator columns of their own, added in the epilogue: a narrow MMA costs what reading its 128 weight rows costs, so one
// MMA twice as wide is cheaper than two (16 tokens, 16,384 x 4,096 gated: 660 cycles of issue per chunk with two).
template <int B_ROWS, int PIECES>
struct LinearTile {
    static constexpr int kN = PIECES * B_ROWS, kSfb = kN > 128 ? 2 : 1;    // operand rows, scale blocks of a chunk
    static constexpr int kCtasPerSm = B_ROWS <= 32 ? 2 : 1;
    // epilogue warps, two or four per tensor-memory lane quadrant, and the converters of DIRECT kernels; a producer and an MMA warp in front
    static constexpr int kConvWarps = B_ROWS <= 32 ? 8 : 16, kThreads = 64 + 32 * kConvWarps;
    static constexpr int kStageBytes = kTileM * 128 + kN * 128 + (1 + kSfb) * kScaleBlockBytes;
    static constexpr int kRedBytes = B_ROWS * kTileM * 4;                  // partial sums of a split K
    static constexpr int kFit = ((kCtasPerSm == 2 ? 111 : 224) * 1024 - kRedBytes) / kStageBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    // tensor memory: the accumulators and, above them, a scale slot per stage - 4 columns of weights, 4 per block of tokens. A stage is filled again
    // only after the MMAs that read it, so its slot's next copies find those MMAs done.
    static constexpr uint32_t kSfStride = 4 + 4 * kSfb, kNeed = kN + kStages * kSfStride;
    static constexpr uint32_t kCols = kNeed <= 64 ? 64 : kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
    static_assert(kStages >= 3 && kNeed <= 512 && kCtasPerSm * kCols <= 512, "too few stages, or more tensor memory than an SM has");
};
template <int B_ROWS, int PIECES>
struct LinearSmem {
    using T = LinearTile<B_ROWS, PIECES>;
    alignas(1024) uint8_t a[T::kStages][kTileM * 128];
    alignas(1024) uint8_t b[T::kStages][T::kN * 128];
    alignas(128) uint8_t sfa[T::kStages][kScaleBlockBytes];
    alignas(128) uint8_t sfb[T::kStages][T::kSfb * kScaleBlockBytes];
    alignas(16) float red[T::kRedBytes / 4];
    uint64_t full[T::kStages], empty[T::kStages], acc_full;
    uint32_t tmem_base, abort_flag;
};
// Eight activations of one row as they lie in memory, and their block's scale byte if they have one. The address is valid
// whatever the place (rows and columns beyond the request read its last row and first columns and are dropped when the values
// are used): with no branch around them, the loads of a whole chunk stay in flight.
template <int PIECES>
struct RawX {
    uint32_t w[PIECES == 2 ? 4 : 2];
    uint32_t scale;
    __device__ __forceinline__ void load(const LinearArgs& p, uint32_t row, uint32_t col) {
        row = row < p.rows ? row : p.rows - 1;
        col = col < p.k ? col : col & (kBlockK - 1);
        const uint64_t at = uint64_t(row) * p.x_pitch + col;
        if constexpr (PIECES == 2) {
            const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + at);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
            scale = 0;
        } else {
            const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.x) + at);
            w[0] = a.x; w[1] = a.y;
            scale = p.x_scales[uint64_t(row) * (p.k / kBlockK) + col / kBlockK];
        }
    }
};

// A converter warp of a DIRECT kernel: eight rows of chunks i, i + kLanes, ... of the request into their stages' token buffers,
// sixteen lanes per row, two rows at a time. What a chunk costs is latency - the loads, then a chain of some twenty dependent
// conversions and shuffles - so the warps work on different chunks and rows, and a warp takes its eight rows without a branch
// (rows beyond the request repeat its last one into the tile's padding). Measured per chunk: 1,160 cycles for eight rows, 2,200
// for sixteen, 3,570 for sixteen with the rows one pair after the other.
template <int B_ROWS, int PIECES>
struct LinearConverter {
    static constexpr uint32_t kStages = LinearTile<B_ROWS, PIECES>::kStages, kParts = B_ROWS / 8;       // kParts warps share a chunk
    static constexpr uint32_t kConvWarps = LinearTile<B_ROWS, PIECES>::kConvWarps;
    // No more chunks at work than there are stages: a warp that has finished chunk i knows chunks up to i - kStages to be consumed,
    // so with a step of at most kStages the parity it waits for next cannot be that of a stage's use before last.
    static constexpr uint32_t kLanes = kConvWarps / kParts < kStages ? kConvWarps / kParts : kStages;
    uint32_t row0, first, g, r0, c0, n_chunks, tok0;
    RawX<PIECES> raw[4];

    __device__ __forceinline__ LinearConverter(uint32_t cw, uint32_t lane, uint32_t c_first, uint32_t chunks, uint32_t token)
        : row0(cw % kParts * 8), first(cw / kParts), g(lane & 15u), r0(row0 + (lane >> 4)), c0(c_first), n_chunks(chunks), tok0(token) {}
    __device__ __forceinline__ void request(const LinearArgs& p, uint32_t i) {
#pragma unroll
        for (int v = 0; v < 4; ++v) raw[v].load(p, tok0 + r0 + 2 * v, (c0 + i) * kChunkK + g * 8);
    }
    template <class Smem>
    __device__ __forceinline__ void run(const LinearArgs& p, Smem& s, uint32_t lane) {
        if (tok0 + row0 >= p.rows || first >= kLanes || first >= n_chunks) return;
        request(p, first);
        for (uint32_t i = first; i < n_chunks; i += kLanes) {
            const uint32_t stage = i % kStages, phase = (i / kStages) & 1u;
            const bool inside = (c0 + i) * kChunkK + g * 8 < p.k;
            if (!__all_sync(0xffffffffu, mbar_wait(&s.empty[stage], phase ^ 1u, &s.abort_flag))) return;
            uint32_t scale[4];
            uint2 hi[4], lo[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const RawX<PIECES>& x = raw[v];
                if constexpr (PIECES == 2) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = inside ? x.w[e] : 0u;
                    const uint32_t amax = block_amax(w, 0xffffffffu);
                    const bool bad = amax >= 0x7f800000u;
                    scale[v] = bad ? 127u : split_scale_byte(amax);
                    split8(w, scale[v], bad, hi[v], lo[v]);
                } else {
                    const bool nan = inside && x.scale == 255u;
                    scale[v] = nan || !inside ? 127u : x.scale;
                    hi[v] = nan ? make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu) : inside ? make_uint2(x.w[0], x.w[1]) : make_uint2(0, 0);
                }
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const uint32_t r = r0 + 2 * v;
                // 128-byte swizzle: 16-byte unit u of row r sits at unit u ^ (r % 8)
                uint8_t* at = s.b[stage] + r * 128 + (((g >> 1) ^ (r & 7u)) << 4) + ((g & 1u) << 3);
                *reinterpret_cast<uint2*>(at) = hi[v];
                if constexpr (PIECES == 2) *reinterpret_cast<uint2*>(at + B_ROWS * 128) = lo[v];
                if ((g & 3u) == 0) {
                    s.sfb[stage][scale_block_offset(int(r), int(g >> 2))] = uint8_t(scale[v]);
                    if constexpr (PIECES == 2) s.sfb[stage][((B_ROWS + r) >> 7) * kScaleBlockBytes + scale_block_offset(int((B_ROWS + r) & 127u), int(g >> 2))] = uint8_t(scale[v] - 4u);
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.full[stage]);
            if (i + kLanes < n_chunks) request(p, i + kLanes);
        }
    }
};

// One CTA: one 128-row weight tile (blockIdx.x >> log_split) x one token tile (blockIdx.y), over its share of the K chunks. The
// 1 << log_split CTAs of a cluster share a tile; they add their partial sums over distributed shared memory in rank order, each
// finishing an equal part of the tile's features, so the result does not depend on timing. Token tiles start on multiples of 128
// (their scale blocks hold 128 tokens): smaller B_ROWS serve requests of at most B_ROWS tokens.
//
// DIRECT (few tokens, or few chunks per CTA; rows on 16-byte boundaries): the epilogue warps, idle while the weights stream, turn the activations of
// each chunk into the pieces in shared memory themselves; no second launch, no workspace. Every weight tile repeats that work, so
// larger requests stage the pieces once (linear_split_kernel) and fetch them with TMA.
template <int B_ROWS, int PIECES, bool GATED, bool DIRECT>
__global__ void __launch_bounds__((LinearTile<B_ROWS, PIECES>::kThreads), (LinearTile<B_ROWS, PIECES>::kCtasPerSm))
linear_w4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TokenMaps maps_x, const LinearArgs p, const uint32_t log_split) {
    using T = LinearTile<B_ROWS, PIECES>;
    using Smem = LinearSmem<B_ROWS, PIECES>;
    extern __shared__ uint8_t smem_raw[];
    Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = 1u << log_split;
    const uint32_t rank = split > 1 ? cluster_ctarank() : 0;
    const uint32_t tile = blockIdx.x >> log_split;
    const uint32_t c0 = p.chunks * rank >> log_split, c1 = p.chunks * (rank + 1) >> log_split;
    const uint32_t tok0 = blockIdx.y * B_ROWS;
    const uint32_t n_valid = p.rows - tok0 < B_ROWS ? p.rows - tok0 : B_ROWS, n_mma = (n_valid + 15) & ~15u;
    volatile uint32_t* abort_flag = &s.abort_flag;

    if (threadIdx.x == 0) {
        const uint32_t filled = DIRECT ? 1 + (n_valid + 7) / 8 : 1;         // the producer, and the converters that share a chunk
        for (int i = 0; i < T::kStages; ++i) { mbar_init(&s.full[i], filled); mbar_init(&s.empty[i], 1); }
        mbar_init(&s.acc_full, 1);
        s.abort_flag = 0;
        mbar_init_fence();
    }
    __syncthreads();
    if (split > 1) cluster_arrive();             // "this CTA has started": its shared memory may be written from now on
    grid_dep_launch();

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (elect_one()) {
            tma_prefetch_desc(&map_w);
            const uint32_t n_chunks = c1 - c0;
            const uint32_t tx = kTileM * 64 + kScaleBlockBytes + (DIRECT ? 0 : PIECES * n_mma * 128 + T::kSfb * kScaleBlockBytes);
            const uint8_t* sfb_g = p.sfb + uint64_t(tok0 >> 7) * p.chunks * T::kSfb * kScaleBlockBytes;
            auto weights = [&](uint32_t i, uint32_t st) {
                const uint32_t c = c0 + i;
                mbar_expect_tx(&s.full[st], tx);
                tma_load_2d(s.a[st], &map_w, int(c * kChunkK), int(tile * kTileM), &s.full[st]);
                bulk_load(s.sfa[st], p.sfa + (uint64_t(tile) * p.chunks + c) * kScaleBlockBytes, kScaleBlockBytes, &s.full[st]);
            };
            // the weights depend on no earlier kernel: their first stages are requested before the stream's last one ends
            const uint32_t early = n_chunks < uint32_t(T::kStages) ? n_chunks : uint32_t(T::kStages);
            for (uint32_t i = 0; i < early; ++i) weights(i, i);
            grid_dep_wait();
            uint32_t stage = 0, phase = 0;
            for (uint32_t i = 0; i < n_chunks; ++i) {
                if (i >= early) {
                    if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort_flag)) { atomicOr(p.fault, uint32_t(kFaultPipeline)); break; }
                    weights(i, stage);
                }
                if constexpr (!DIRECT) {
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
                    bulk_load(s.sfb[stage], sfb_g + uint64_t(c) * T::kSfb * kScaleBlockBytes, T::kSfb * kScaleBlockBytes, &s.full[stage]);
                }
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
        tmem_alloc(&s.tmem_base, T::kCols);      // while the first loads are under way; the epilogue warps learn the address below
        tmem_relinquish();
        tc_fence_before();
        named_bar_sync(1, 32 + 32 * T::kConvWarps);
        tc_fence_after();
        const uint32_t tb = s.tmem_base;
        grid_dep_wait();                         // bounded waits start when the stream's earlier kernels have ended, however long they take
        if (elect_one()) {
            const uint32_t idesc0 = idesc_mx(kFmtE2M1, kFmtE4M3, (PIECES - 1) * B_ROWS + n_mma, 0, 0);
            const uint64_t a_desc0 = desc_sw128(smem_u32(s.a[0])), b_desc0 = desc_sw128(smem_u32(s.b[0]));
            const uint64_t sfa_desc0 = desc_scale_block(smem_u32(s.sfa[0])), sfb_desc0 = desc_scale_block(smem_u32(s.sfb[0]));
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t c = c0; c < c1; ++c) {
                if (!mbar_wait(&s.full[stage], phase, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t t_sf = tb + T::kN + stage * T::kSfStride;
                tc_cp_scales(t_sf, sfa_desc0 + stage * (sizeof(s.sfa[0]) >> 4));
#pragma unroll
                for (int b = 0; b < T::kSfb; ++b) tc_cp_scales(t_sf + 4 + 4 * b, sfb_desc0 + stage * (sizeof(s.sfb[0]) >> 4) + b * (kScaleBlockBytes >> 4));
                const uint64_t ad = a_desc0 + stage * (sizeof(s.a[0]) >> 4), bd = b_desc0 + stage * (sizeof(s.b[0]) >> 4);
#pragma unroll
                for (uint32_t kb = 0; kb < 4; ++kb)
                    tc_mma_mx(tb, ad + 2 * kb, bd + 2 * kb, idesc0 | (kb << 4) | (kb << 29), t_sf, t_sf + 4, (c != c0 || kb) ? 1u : 0u);
                tc_commit(&s.empty[stage]);
                if (++stage == uint32_t(T::kStages)) { stage = 0; phase ^= 1u; }
            }
            if (ok) tc_commit(&s.acc_full);
            else atomicOr(p.fault, uint32_t(kFaultPipeline));
        }
        __syncwarp();
        if (split > 1) cluster_wait();
    } else {
        named_bar_sync(1, 32 + 32 * T::kConvWarps);
        tc_fence_after();
        const uint32_t tb = s.tmem_base;
        grid_dep_wait();                         // as the MMA warp; and the activations come from the stream's earlier kernels
        if constexpr (DIRECT) {
            LinearConverter<B_ROWS, PIECES> conv(uint32_t(warp - 2), uint32_t(lane), c0, c1 - c0, tok0);
            conv.run(p, s, uint32_t(lane));
        }
        // ------------------------------------------------------------ epilogue, first half: tensor memory -> where it is added
        const uint32_t q = uint32_t(warp) & 3u;            // lane quadrant; the quadrant's warps take sixteen tokens in turn
        const uint32_t row = q * 32u + lane;               // weight row of the tile
        const bool ok = acc_wait(&s.acc_full, 0, abort_flag, p);
        __syncwarp();
        if (split > 1) cluster_wait();
        if (__all_sync(0xffffffffu, ok)) {
            tc_fence_after();
            const uint32_t t_acc = tb + ((q * 32u) << 16);
            // owner of a row and its place there: features are dealt in equal runs, gate and up of a feature together
            const uint32_t log_run = (GATED ? 6 : 7) - log_split, f = GATED ? q * 16 + (lane & 15) : row;
            const uint32_t owner = f >> log_run, slot = (f & ((1u << log_run) - 1)) + (GATED ? uint32_t(lane >> 4) << log_run : 0);
            const uint32_t base = (split > 1 ? cluster_map(smem_u32(s.red), owner) : smem_u32(s.red)) + slot * 4;
            const uint32_t feat = tile * (GATED ? 64 : kTileM) + f;
            for (uint32_t col = uint32_t(warp - 2) / 4 * 16; col < n_mma; col += T::kConvWarps * 4) {
                uint32_t r[16];
                tmem_ld16(t_acc + col, r);
                if constexpr (PIECES == 2) {
                    uint32_t l[16];
                    tmem_ld16(t_acc + B_ROWS + col, l);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(l[j]));
                } else {
                    tmem_wait_ld();
                }
                if (split == 1) {
                    store_columns<GATED>(p, r, tok0 + col, tok0 + n_valid, feat, lane);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (col + j < n_valid) st_cluster_f32(base + (((rank * n_valid + col + j) << (7 - log_split)) << 2), __uint_as_float(r[j]));
                }
            }
            tc_fence_before();
        }
    }
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    if (split > 1) {
        // -------------------------------------------------------- epilogue, second half: partial sums in rank order
        const uint32_t log_feats = (GATED ? 6 : 7) - log_split, feats = 1u << log_feats;
        const uint32_t feat0 = tile * (GATED ? 64 : kTileM) + rank * feats;
        for (uint32_t i = threadIdx.x; i < n_valid << log_feats; i += T::kThreads) {
            const uint32_t f = i & (feats - 1), col = i >> log_feats;
            if (feat0 + f >= p.n) continue;
            const float* from = s.red + (col << (7 - log_split)) + f;
            float v = 0.0f, u = 0.0f;
            for (uint32_t r = 0; r < split; ++r, from += n_valid << (7 - log_split)) {
                v += from[0];
                if constexpr (GATED) u += from[feats];
            }
            store_y(p, tok0 + col, feat0 + f, GATED ? silu_gate(v, u) : v);
        }
    }
    if (warp == 1) tmem_dealloc(s.tmem_base, T::kCols);
}

// ---- the product on CTA pairs (prefill) -----------------------------------------------------------------------------
// cta_group::2: two CTAs of a cluster run one MMA of M = 256 (128 weight rows each) x N = `tile` tokens (at most 256 with one piece, 224
// with two), half of the token rows in each CTA's shared memory. What bounds a block-scaled MMA at prefill is shared memory, which feeds the
// operands (128 B/clk) and takes the loads: per 128-wide chunk and CTA, 224 tokens of two pieces read 60 KB and fill 44 KB in 896 cycles
// of math, 119 B/clk; 128 tokens wide it would be 160, a single CTA of 128 x 128 tokens 224.
// Each piece has accumulator columns of its own, added once in the epilogue. The tensor core truncates its running sum to FP32 after every
// MMA. The leading pieces' products lie on a coarse grid, so that little falls off; with the second pieces' sixteen times finer
// products in the same column every step loses a part of a unit in the last place, towards zero (2,048 tokens, 4,096 x 4,096, FP32
// out: off by 8.8e-7 of the result with shared columns). Two sets of 224 columns leave 64 to the scales.
// The accumulators are pulled into registers (64 per thread) and handed back before the epilogue's math, so that the next
// item's MMAs run meanwhile. Barriers as in gemm_mx_pair.cuh: loads of both CTAs report to the first CTA's `full`.
constexpr uint32_t kLpMaxTokens = 256;
constexpr int kLpEpiWarps = 16, kLpThreads = 64 + 32 * kLpEpiWarps;
template <int PIECES>
struct LinearPairTile {
    static constexpr uint32_t kTokens = PIECES == 2 ? 224 : kLpMaxTokens;       // widest token tile; a piece's accumulator columns
    // scale slots above the accumulators: 4 columns of weights, 8 per piece of tokens, one per stage or as many as there is room for
    static constexpr uint32_t kStages = PIECES == 2 ? 4 : 6, kSf = PIECES * kTokens, kSfStride = 4 + 8 * PIECES;
    static constexpr uint32_t kSfRoom = (kTmemCols - kSf) / kSfStride, kSfSlots = kSfRoom < kStages ? kSfRoom : kStages;
    static_assert(kSfSlots >= 3, "two chunks' MMAs at work while a third's scales are copied");
};

struct LinearPairMaps {
    CUtensorMap w;          // weight rows, box 128
    CUtensorMap tok[5];     // token rows, boxes of 128 / 64 / 32 / 16 / 8
    CUtensorMap sfa;        // weight scale blocks as rows of 128 u32, box 1
    CUtensorMap sfb;        // token scale blocks, box: those of a tile's chunk
};
template <int PIECES>
struct LinearPairSmem {
    static constexpr uint32_t kStages = LinearPairTile<PIECES>::kStages;
    static constexpr uint32_t kPieceBytes = LinearPairTile<PIECES>::kTokens / 2 * 128;
    alignas(1024) uint8_t a[kStages][kTileM * 128];
    alignas(1024) uint8_t b[kStages][PIECES * kPieceBytes];
    alignas(128) uint8_t sfa[kStages][kScaleBlockBytes];
    alignas(128) uint8_t sfb[kStages][2 * PIECES * kScaleBlockBytes];       // [128-token run of the tile][piece]
    uint64_t full[kStages], empty[kStages], acc_full, acc_empty;
    uint32_t tmem_base, abort_flag;
};
static_assert(sizeof(LinearPairSmem<2>) + 1024 <= 232448 && sizeof(LinearPairSmem<1>) + 1024 <= 232448, "a CTA has at most 227 KB of shared memory");

// Items: 256 image rows x `tile` tokens, the weight rows running fastest, strided over the pairs of the grid.
template <int PIECES, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kLpThreads, 1)
linear_pair_kernel(const __grid_constant__ LinearPairMaps maps, const LinearArgs p, const uint32_t m_pairs, const uint32_t n_items, const uint32_t tile_n) {
    using Smem = LinearPairSmem<PIECES>;
    using T = LinearPairTile<PIECES>;
    constexpr uint32_t kStages = Smem::kStages;
    extern __shared__ uint8_t smem_raw[];
    Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    volatile uint32_t* abort_flag = &s.abort_flag;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kStages; ++i) { mbar_init(&s.full[i], 1); mbar_init(&s.empty[i], 1); }
        mbar_init(&s.acc_full, 1);
        mbar_init(&s.acc_empty, 2 * kLpEpiWarps);
        s.abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) { tmem_alloc_pair(&s.tmem_base, kTmemCols); tmem_relinquish_pair(); }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();          // the partner's barriers exist before anything arrives on them
    tc_fence_after();
    grid_dep_launch();
    const uint32_t tb = s.tmem_base;
    const auto tile_tokens = [&](uint32_t t) { const uint32_t left = p.rows - t * tile_n; return left < tile_n ? left : tile_n; };
    const uint32_t runs = tile_n > 128 ? 2 : 1;          // 128-token runs of a tile, one scale block each per piece

    if (warp == 0) {
        // ------------------------------------------------------------ producer (both CTAs)
        if (elect_one()) {
            tma_prefetch_desc(&maps.w);
            uint32_t stage = 0, phase = 0, issued = 0;
            bool ok = true;
            for (uint32_t it = pair_id; it < n_items && ok; it += n_pairs) {
                const uint32_t m = it % m_pairs, t = it / m_pairs;
                const uint32_t n_mma = (tile_tokens(t) + 15) & ~15u, half = n_mma >> 1;
                const uint32_t tile = 2 * m + rank;
                const uint32_t tx = kTileM * 64 + PIECES * half * 128 + kScaleBlockBytes + runs * PIECES * kScaleBlockBytes;
                const auto weights = [&](uint32_t c, uint32_t st) {
                    const uint32_t bar = cluster_map(smem_u32(&s.full[st]), 0);
                    if (rank == 0) mbar_expect_tx(&s.full[st], 2 * tx);        // the bytes of both CTAs' loads
                    tma_load_2d_pair(s.a[st], &maps.w, int(c * kChunkK), int(tile * kTileM), bar);
                    tma_load_2d_pair(s.sfa[st], &maps.sfa, 0, int(tile * p.chunks + c), bar);
                };
                // the weights depend on no earlier kernel: the first stages' are requested before the stream's last one ends
                uint32_t early = 0;
                if (it == pair_id) {
                    early = p.chunks < kStages ? p.chunks : kStages;
                    for (uint32_t c = 0; c < early; ++c) weights(c, c);
                    grid_dep_wait();
                }
                for (uint32_t c = 0; c < p.chunks; ++c) {
                    if (c >= early) {
                        if (!mbar_wait(&s.empty[stage], phase ^ 1u, abort_flag)) { ok = false; break; }
                        weights(c, stage);
                    }
                    const uint32_t bar = cluster_map(smem_u32(&s.full[stage]), 0);
#pragma unroll
                    for (uint32_t piece = 0; piece < PIECES; ++piece) {
                        uint32_t r = 0;
#pragma unroll
                        for (uint32_t b = 0; b < 5; ++b) {
                            const uint32_t box = 128u >> b;
                            if (half - r >= box) {
                                tma_load_2d_pair(s.b[stage] + piece * Smem::kPieceBytes + r * 128, &maps.tok[b], int(c * kChunkK),
                                                 int(piece * p.rows_cap + t * tile_n + rank * half + r), bar);
                                r += box;
                            }
                        }
                    }
                    tma_load_2d_pair(s.sfb[stage], &maps.sfb, 0, int((t * p.chunks + c) * runs * PIECES), bar);
                    ++issued;
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
            if (!ok) atomicOr(p.fault, uint32_t(kFaultPipeline));
            if (*abort_flag && rank == 0) {        // a wait ran out: give the loads under way time to land
                const long long t0 = clock64();
                for (uint32_t i = 0; i < kStages && i < issued; ++i)
                    while (!mbar_try_wait(&s.full[i], phase ^ (i < stage ? 0u : 1u)) && clock64() - t0 < kWaitCycles) {}
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issue (first CTA of the pair only)
        grid_dep_wait();             // bounded waits start when the stream's earlier kernels have ended, however long they take
        if (rank == 0 && elect_one()) {
            uint32_t stage = 0, phase = 0, local = 0, slot = 0;
            uint32_t issued = 0, old_stage = 0, old_phase = 0;       // chunks issued; the one whose scale slot comes next
            bool ok = true;
            const uint64_t a_desc0 = desc_sw128(smem_u32(s.a[0])), b_desc0 = desc_sw128(smem_u32(s.b[0]));
            const uint64_t sfa_desc0 = desc_scale_block(smem_u32(s.sfa[0])), sfb_desc0 = desc_scale_block(smem_u32(s.sfb[0]));
            for (uint32_t it = pair_id; it < n_items && ok; it += n_pairs, ++local) {
                const uint32_t n_mma = (tile_tokens(it / m_pairs) + 15) & ~15u;
                const uint32_t idesc0 = idesc_mx_pair(kFmtE2M1, kFmtE4M3, n_mma, 0, 0);
                if (!mbar_wait(&s.acc_empty, (local & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                tc_fence_after();
                for (uint32_t c = 0; c < p.chunks; ++c) {
                    if (!mbar_wait(&s.full[stage], phase, abort_flag)) { ok = false; break; }
                    if constexpr (T::kSfSlots < kStages) {
                        // with fewer slots than stages a refilled stage does not yet say that the slot's last MMAs are done: their commit does
                        if (issued >= T::kSfSlots) {
                            if (!mbar_wait(&s.empty[old_stage], old_phase, abort_flag)) { ok = false; break; }
                            if (++old_stage == kStages) { old_stage = 0; old_phase ^= 1u; }
                        }
                        ++issued;
                    }
                    tc_fence_after();
                    const uint32_t t_sf = tb + T::kSf + slot * T::kSfStride;
                    if (++slot == T::kSfSlots) slot = 0;
                    tc_cp_scales_pair(t_sf, sfa_desc0 + stage * (sizeof(s.sfa[0]) >> 4));
                    const uint64_t sfb_d = sfb_desc0 + stage * (sizeof(s.sfb[0]) >> 4);
#pragma unroll
                    for (uint32_t piece = 0; piece < PIECES; ++piece) {
                        tc_cp_scales_pair(t_sf + 4 + 8 * piece, sfb_d + piece * (kScaleBlockBytes >> 4));
                        if (runs == 2) tc_cp_scales_pair(t_sf + 8 + 8 * piece, sfb_d + (PIECES + piece) * (kScaleBlockBytes >> 4));
                    }
                    const uint64_t ad = a_desc0 + stage * (sizeof(s.a[0]) >> 4), bd = b_desc0 + stage * (sizeof(s.b[0]) >> 4);
#pragma unroll
                    for (uint32_t piece = 0; piece < PIECES; ++piece)
#pragma unroll
                        for (uint32_t kb = 0; kb < 4; ++kb)
                            tc_mma_mx_pair(tb + piece * T::kTokens, ad + 2 * kb, bd + piece * (Smem::kPieceBytes >> 4) + 2 * kb, idesc0 | (kb << 4) | (kb << 29),
                                           t_sf, t_sf + 4 + 8 * piece, (c | kb) ? 1u : 0u);
                    tc_commit_pair(&s.empty[stage]);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
                if (ok) tc_commit_pair(&s.acc_full);
            }
            if (!ok) atomicOr(p.fault, uint32_t(kFaultPipeline));
        }
    } else {
        // ------------------------------------------------------------ epilogue (both CTAs)
        const uint32_t q = uint32_t(warp) & 3u, col0 = uint32_t(warp - 2) / 4 * 64;      // lane quadrant, first of the warp's 64 tokens
        const uint32_t t_acc = tb + ((q * 32u) << 16) + col0;
        grid_dep_wait();             // as the MMA warp
        uint32_t local = 0;
        for (uint32_t it = pair_id; it < n_items; it += n_pairs, ++local) {
            const uint32_t m = it % m_pairs, t = it / m_pairs, n_valid = tile_tokens(t), n_mma = (n_valid + 15) & ~15u;
            const bool got = __all_sync(0xffffffffu, acc_wait(&s.acc_full, local & 1u, abort_flag, p));
            if (!got && __any_sync(0xffffffffu, *abort_flag != 0)) break;        // the pipeline stands still
            tc_fence_after();
            uint32_t r[4][16];
#pragma unroll
            for (uint32_t g = 0; g < 4; ++g)
                if (col0 + 16 * g < n_mma) tmem_ld16(t_acc + 16 * g, r[g]);
            if constexpr (PIECES == 2) {
#pragma unroll
                for (uint32_t g = 0; g < 4; ++g) {
                    if (col0 + 16 * g >= n_mma) continue;
                    uint32_t l[16];
                    tmem_ld16(t_acc + T::kTokens + 16 * g, l);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) r[g][j] = __float_as_uint(__uint_as_float(r[g][j]) + __uint_as_float(l[j]));
                }
            }
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(cluster_map(smem_u32(&s.acc_empty), 0));
            if (!got) continue;
            const uint32_t tile = 2 * m + rank, feat = GATED ? tile * 64 + q * 16 + (lane & 15) : tile * kTileM + q * 32 + lane;
#pragma unroll
            for (uint32_t g = 0; g < 4; ++g)
                if (col0 + 16 * g < n_valid) store_columns<GATED>(p, r[g], t * tile_n + col0 + 16 * g, t * tile_n + n_valid, feat, lane);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();          // nothing of either CTA is torn down while the partner may still signal it
    if (warp == 1) tmem_dealloc_pair(tb, kTmemCols);
}

}  // namespace m26b
