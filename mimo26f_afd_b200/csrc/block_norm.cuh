// The step between two blocks of a decoder, one pass over each row:
//     u = y_0 + y_1 + ... (rank order)          the block's output, one BF16 plane per rank or one FP32 plane
//     u = u / sqrt(mean(u^2) + eps) * post_w    norm after the block (optional)
//     h = residual_scale * residual + y_scale * gate * u
//     n = h / sqrt(mean(h^2) + eps) * pre_w     norm before the next block (optional)
// The reference runs it as three launches on the coordinator (rank sum, h += f, rmsnorm:
// crates/mimo26-coordinator/kernels/glue.cu:55-59, 200-213); the operands of a row are read once here and the row stays
// in registers between the two reductions. Everything is FP32 from the loads to the single rounding of each output.
//
// What bounds it: HBM traffic (planes + residual in, h and n out); about twelve operations per element. Measured (BF16 plane, post
// and pre norm): 8,192 x 4,096 with an FP32 residual stream 75 us = 5.4 TB/s, BF16 stream and a gate per element 61 us = 5.5 TB/s,
// 8,192 x 4,095 dense rows 95 us = 4.2 TB/s, one row 3.5 us. Issue slots matter next: the row's shared factors are folded into one,
// the root is rsqrtf, and what differs from call to call is asked per vector or per four elements.
// Layout: rows on vector boundaries stay in registers (block_norm_kernel: a row belongs to a warp or a CTA, a thread owns PER
// vectors of VEC elements, a row's worth apart, so that every access of a warp is one contiguous run); other and wider rows wait for
// their reductions in shared memory (block_norm_any_kernel).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include <type_traits>

#include "sm100_ptx.cuh"

namespace m26b {

enum { kGateNone = 0, kGateToken = 1, kGateChannel = 2, kGateElement = 3 };

struct NormArgs {
    const void* y[8];
    int planes;                 // 0: no block output
    int y_f32, h_f32, n_f32, w_f32;
    uint64_t y_pitch, h_pitch, n_pitch;     // elements
    const void *post_w, *gate, *residual, *pre_w;
    int gate_kind;
    float y_scale, residual_scale, eps, inv_width;      // y_scale 1 without planes, residual_scale 0 without a residual
    uint32_t rows, width;
    void *h_out, *n_out;
};

// VEC consecutive elements starting at element `i`, of which `left` belong to the row. VEC 8: 16-byte aligned, always whole. VEC 4:
// 8-byte (BF16) or 16-byte (FP32) aligned; a row's last vector may be short, and nothing beyond the row is touched.
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float load_one(const void* base, int f32, uint64_t i) {
    return f32 ? static_cast<const float*>(base)[i] : __uint_as_float(uint32_t(static_cast<const uint16_t*>(base)[i]) << 16);
}
template <int VEC>
__device__ __forceinline__ void load_elems(const void* base, int f32, uint64_t i, float (&v)[VEC], uint32_t left = VEC) {
    if constexpr (VEC == 4) {
        if (left < 4) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] = e < left ? load_one(base, f32, i + e) : 0.0f;
        } else if (f32) {
            const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        } else {
            const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
            v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
        }
    } else if (f32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
        const float4 a = p[0], b = p[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = bf16_lo(w[j]); v[2 * j + 1] = bf16_hi(w[j]); }
    }
}
// Two floats as BF16 (nearest even, NaN kept), the first in the low half.
__device__ __forceinline__ uint32_t bf16x2_rn(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void store_one(void* base, int f32, uint64_t i, float v) {
    if (f32) static_cast<float*>(base)[i] = v;
    else static_cast<uint16_t*>(base)[i] = uint16_t(bf16x2_rn(v, 0.0f));
}
template <int VEC>
__device__ __forceinline__ void store_elems(void* base, int f32, uint64_t i, const float (&v)[VEC], uint32_t left = VEC) {
    if constexpr (VEC == 4) {
        if (left < 4) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (e < left) store_one(base, f32, i + e, v[e]);
        } else if (f32) {
            *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) = make_uint2(bf16x2_rn(v[0], v[1]), bf16x2_rn(v[2], v[3]));
        }
    } else if (f32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) =
            make_uint4(bf16x2_rn(v[0], v[1]), bf16x2_rn(v[2], v[3]), bf16x2_rn(v[4], v[5]), bf16x2_rn(v[6], v[7]));
    }
}

struct OpSum { __device__ static float f(float a, float b) { return a + b; } };
struct OpMax { __device__ static float f(float a, float b) { return fmaxf(a, b); } };
// Reduction over the row's threads: the warp, or (BLOCK) all warps of the CTA through `slots` (32 floats; one array per use).
template <class Op, bool BLOCK>
__device__ __forceinline__ float row_reduce(float v, float* slots) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = Op::f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (BLOCK) {
        const int warps = int(blockDim.x) >> 5;
        if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
        __syncthreads();
        const int lane = int(threadIdx.x & 31);
        v = slots[lane < warps ? lane : 0];
        if (lane >= warps) v = 0.0f;                 // neutral for the sum, and for the maximum of magnitudes
#pragma unroll
        for (int o = 16; o; o >>= 1) v = Op::f(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}
// 1 / sqrt(mean(v^2) + eps) over the row. A sum of squares that leaves FP32 (values above 2^63) is taken again of the
// row divided by a power of two near its largest magnitude; rows that hold an infinity or a NaN keep what FP32 gives.
template <int E, bool BLOCK>
__device__ __forceinline__ float row_rrms(const float (&v)[E], float inv_width, float eps, float (*slots)[32]) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(v[e], v[e], ss);
    ss = row_reduce<OpSum, BLOCK>(ss, slots[0]);
    if (__builtin_expect(!(ss < __int_as_float(0x7f800000)), 0)) {      // the same answer in every thread of the row
        float big = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) big = fmaxf(big, fabsf(v[e]));
        big = row_reduce<OpMax, BLOCK>(big, slots[1]);
        if (big < __int_as_float(0x7f800000) && ss == ss) {
            const float down = 0x1p-100f;                                // |v| <= 2^128: squares at most 2^56
            float s2 = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) { const float a = v[e] * down; s2 = fmaf(a, a, s2); }
            s2 = row_reduce<OpSum, BLOCK>(s2, slots[2]);
            return down * rsqrtf(s2 * inv_width);                        // eps * 2^-200 is nothing beside s2 >= 2^-74
        }
    }
    return rsqrtf(fmaf(ss, inv_width, eps));
}

// Whether the factors of u that a row shares - y_scale, the token's gate, 1 / rms - may be folded into one, so that u meets them in one
// multiplication per element. Not where FP32 does not hold their product well (rows of 1e38 and a scale of 1e-6: 1e-44, three bits): then
// 1 / rms and the gate are applied to the row first. Asked once per row (8,192 x 4,096 BF16 60.8 -> 61.7 us; a branch per vector 73.9).
__device__ __forceinline__ bool foldable(float product) { return fabsf(product) > 0x1p-32f && fabsf(product) < 0x1p32f; }

// VEC elements as they lie in memory: loads are issued for a whole row before anything waits for one of them.
template <int VEC, bool F32>
struct RawVec {
    uint32_t w[VEC * (F32 ? 4 : 2) / 4];
    __device__ __forceinline__ void load(const void* base, uint64_t i, uint32_t left = VEC) {
        if constexpr (VEC == 4) {
            if (left < 4) {
                zero();
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (e < left) {
                        if constexpr (F32) w[e] = static_cast<const uint32_t*>(base)[i + e];
                        else w[e / 2] |= uint32_t(static_cast<const uint16_t*>(base)[i + e]) << (16 * (e & 1));
                    }
            } else if constexpr (F32) {
                const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
            } else {
                const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i);
                w[0] = a.x; w[1] = a.y;
            }
        } else {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + i * (F32 ? 4 : 2));
#pragma unroll
            for (int q = 0; q < VEC * (F32 ? 4 : 2) / 16; ++q) { const uint4 a = p[q]; w[4 * q] = a.x; w[4 * q + 1] = a.y; w[4 * q + 2] = a.z; w[4 * q + 3] = a.w; }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (uint32_t& v : w) v = 0;
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (F32) return __uint_as_float(w[e]);
        else return __uint_as_float((e & 1) ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
};

// A row belongs to a warp (THREADS 32: four rows per CTA) or to a CTA; both stride over the rows by the grid, and the next row's
// operands are requested before this row's reductions are waited for. Y32 / H32: FP32 planes / residual stream. GATE_ELEM: a gate per element.
// Elements a thread owns beyond the row's end are zero in u and h before each reduction and are never stored.
template <int VEC, int PER, int THREADS, bool Y32, bool H32, bool GATE_ELEM>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS) block_norm_kernel(const NormArgs p) {
    constexpr bool BLOCK = THREADS > 32;
    constexpr int E = PER * VEC;
    __shared__ float slots_all[2][6][32];
    constexpr uint32_t threads = THREADS;              // of a row; a constant, so that a thread's vectors are one address and offsets
    const uint32_t t = BLOCK ? threadIdx.x : threadIdx.x & 31u;
    const uint32_t rows_at_once = BLOCK ? gridDim.x : gridDim.x * 4;
    uint32_t row = BLOCK ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
    RawVec<VEC, Y32> ry[PER], rg[PER];
    RawVec<VEC, H32> rh[PER];
    const bool has_y = p.planes > 0, has_h = p.residual != nullptr;
    const auto request = [&](uint32_t r) {
        const uint64_t yo = uint64_t(r) * p.y_pitch, ho = uint64_t(r) * p.h_pitch;
        if (has_y)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if ((t + j * threads) * VEC < p.width) ry[j].load(p.y[0], yo + (t + j * threads) * VEC, p.width - (t + j * threads) * VEC);
        if (has_h)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if ((t + j * threads) * VEC < p.width) rh[j].load(p.residual, ho + (t + j * threads) * VEC, p.width - (t + j * threads) * VEC);
        if (GATE_ELEM)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if ((t + j * threads) * VEC < p.width) rg[j].load(p.gate, yo + (t + j * threads) * VEC, p.width - (t + j * threads) * VEC);
    };
#pragma unroll
    for (int j = 0; j < PER; ++j) { ry[j].zero(); rh[j].zero(); rg[j].zero(); }
    grid_dep_wait();                                 // the block's output comes from the stream's earlier kernels
    grid_dep_launch();
    if (row < p.rows) request(row);
    for (uint32_t turn = 0; row < p.rows; row += rows_at_once, ++turn) {
        float (*slots)[32] = slots_all[turn & 1];    // the other set may still be read by slower warps of the row before
        const uint64_t yo = uint64_t(row) * p.y_pitch, ho = uint64_t(row) * p.h_pitch, no = uint64_t(row) * p.n_pitch;
        float u[E], h[E];
        RawVec<VEC, Y32> cg[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            cg[j] = rg[j];
#pragma unroll
            for (int e = 0; e < VEC; ++e) { u[j * VEC + e] = ry[j].get(e); h[j * VEC + e] = rh[j].get(e); }
        }
        // further planes, two at a time, every load of the two issued before the first is used
#pragma unroll
        for (int q = 1; q < 8; q += 2) {
            if (q >= p.planes) break;
            RawVec<VEC, Y32> more[2][PER];
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int j = 0; j < PER; ++j) more[z][j].zero();
#pragma unroll
            for (int z = 0; z < 2; ++z)
                if (q + z < p.planes)
#pragma unroll
                    for (int j = 0; j < PER; ++j)
                        if ((t + j * threads) * VEC < p.width) more[z][j].load(p.y[q + z], yo + (t + j * threads) * VEC, p.width - (t + j * threads) * VEC);
#pragma unroll
            for (int z = 0; z < 2; ++z)
                if (q + z < p.planes)
#pragma unroll
                    for (int j = 0; j < PER; ++j)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) u[j * VEC + e] += more[z][j].get(e);
        }
        if (rows_at_once < p.rows - row) request(row + rows_at_once);
        float r1 = p.y_scale, rrms = 1.0f;             // r1: every factor of u that the row shares
        if (p.gate_kind == kGateToken) r1 *= static_cast<const float*>(p.gate)[row];
        if (p.post_w) { rrms = row_rrms<E, BLOCK>(u, p.inv_width, p.eps, slots); r1 *= rrms; }
        if (__builtin_expect(!foldable(r1), 0)) {
            const float gate = p.gate_kind == kGateToken ? static_cast<const float*>(p.gate)[row] : 1.0f;
            r1 = p.y_scale;
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] = u[e] * rrms * gate;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = (t + j * threads) * VEC;
            if (i >= p.width) continue;
            float a[VEC], w[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = u[j * VEC + e] * r1;
            if (p.post_w) {
                load_elems<VEC>(p.post_w, p.w_f32, i, w, p.width - i);
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= w[e];
            }
            if (GATE_ELEM) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= cg[j].get(e);
            } else if (p.gate_kind == kGateChannel) {
                load_elems<VEC>(p.gate, p.w_f32, i, w, p.width - i);
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= w[e];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = fmaf(h[j * VEC + e], p.residual_scale, a[e]);
            if (p.h_out) store_elems<VEC>(p.h_out, H32, ho + i, a, p.width - i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[j * VEC + e] = a[e];
        }
        if (!p.n_out) continue;
        const float r2 = row_rrms<E, BLOCK>(h, p.inv_width, p.eps, slots + 3);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = (t + j * threads) * VEC;
            if (i >= p.width) continue;
            float a[VEC], w[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = h[j * VEC + e] * r2;
            if (p.pre_w) {
                load_elems<VEC>(p.pre_w, p.w_f32, i, w, p.width - i);
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= w[e];
            }
            store_elems<VEC>(p.n_out, p.n_f32, no + i, a, p.width - i);
        }
    }
}

// ---- rows on any boundary ------------------------------------------------------------------------------------------------
// The same step element by element: a thread's elements are blockDim apart, four of them at a time, and the row waits for the two
// reductions in shared memory (FP32) instead of in registers, so that many rows are in flight per SM and their latencies cover
// each other. What differs from call to call is asked once per four elements: uniform branches around every element cost more
// than the element.
__device__ __forceinline__ float row_rrms_shared(float ss, const float* row, uint32_t width, float inv_width, float eps, float (*slots)[32]) {
    ss = row_reduce<OpSum, true>(ss, slots[0]);
    if (__builtin_expect(!(ss < __int_as_float(0x7f800000)), 0)) {             // as row_rrms
        float big = 0.0f, s2 = 0.0f;
        for (uint32_t i = threadIdx.x; i < width; i += blockDim.x) {
            const float a = row[i] * 0x1p-100f;
            big = fmaxf(big, fabsf(row[i]));
            s2 = fmaf(a, a, s2);
        }
        big = row_reduce<OpMax, true>(big, slots[1]);
        s2 = row_reduce<OpSum, true>(s2, slots[2]);
        if (big < __int_as_float(0x7f800000) && ss == ss) return 0x1p-100f * rsqrtf(s2 * inv_width);
    }
    return rsqrtf(fmaf(ss, inv_width, eps));
}
template <uint32_t T, bool Y32, bool H32>
__global__ void __launch_bounds__(T, 2048 / T) block_norm_any_kernel(const NormArgs p) {
    extern __shared__ float row_mem[];
    __shared__ float slots_all[2][6][32];
    const uint32_t t = threadIdx.x;
    const bool has_h = p.residual != nullptr;
    // f(first element, how many of the four at distance T there are); all four whenever they fit, which is a constant then
    const auto four = [&](auto&& f) {
        uint32_t i = t;
        for (; i + 3 * T < p.width; i += 4 * T) f(i, std::integral_constant<uint32_t, 4>{});
        if (i < p.width) f(i, std::integral_constant<uint32_t, 0>{});
    };
    grid_dep_wait();                                 // the block's output comes from the stream's earlier kernels
    grid_dep_launch();
    uint32_t turn = 0;
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x, ++turn) {
        float (*slots)[32] = slots_all[turn & 1];    // the other set may still be read by slower warps of the row before
        const uint64_t yo = row * p.y_pitch, ho = row * p.h_pitch, no = row * p.n_pitch;
        float r1 = p.y_scale, rrms = 1.0f;             // r1: every factor of u that the row shares
        if (p.gate_kind == kGateToken) r1 *= static_cast<const float*>(p.gate)[row];
        float ss = 0.0f;
        four([&](uint32_t i, auto full) {
            constexpr bool kAll = decltype(full)::value == 4;
            float u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
            for (int q = 0; q < p.planes; ++q) {
                float b[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) b[e] = kAll || i + e * T < p.width ? load_one(p.y[q], Y32, yo + i + e * T) : 0.0f;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) u[e] = q ? u[e] + b[e] : b[e];
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                ss = fmaf(u[e], u[e], ss);
                if (kAll || i + e * T < p.width) row_mem[i + e * T] = u[e];
            }
        });
        if (p.post_w) { rrms = row_rrms_shared(ss, row_mem, p.width, p.inv_width, p.eps, slots); r1 *= rrms; }
        if (__builtin_expect(!foldable(r1), 0)) {
            const float gate = p.gate_kind == kGateToken ? static_cast<const float*>(p.gate)[row] : 1.0f;
            r1 = p.y_scale;
            for (uint32_t i = t; i < p.width; i += T) row_mem[i] = row_mem[i] * rrms * gate;
        }
        ss = 0.0f;
        four([&](uint32_t i, auto full) {
            constexpr bool kAll = decltype(full)::value == 4;
            float h[4] = {0.0f, 0.0f, 0.0f, 0.0f}, w[4], a[4];
            if (has_h)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) h[e] = kAll || i + e * T < p.width ? load_one(p.residual, H32, ho + i + e * T) : 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) a[e] = kAll || i + e * T < p.width ? row_mem[i + e * T] * r1 : 0.0f;
            const auto times = [&](const void* base, int f32, uint64_t first) {
                if (f32) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) w[e] = kAll || i + e * T < p.width ? load_one(base, 1, first + i + e * T) : 0.0f;
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) w[e] = kAll || i + e * T < p.width ? load_one(base, 0, first + i + e * T) : 0.0f;
                }
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) a[e] *= w[e];
            };
            if (p.post_w) times(p.post_w, p.w_f32, 0);
            if (p.gate_kind == kGateElement) times(p.gate, Y32, yo);
            else if (p.gate_kind == kGateChannel) times(p.gate, p.w_f32, 0);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                h[e] = fmaf(h[e], p.residual_scale, a[e]);
                if (kAll || i + e * T < p.width) {
                    ss = fmaf(h[e], h[e], ss);
                    row_mem[i + e * T] = h[e];
                }
            }
            if (p.h_out) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (kAll || i + e * T < p.width) store_one(p.h_out, H32, ho + i + e * T, h[e]);
            }
        });
        if (!p.n_out) continue;
        const float r2 = row_rrms_shared(ss, row_mem, p.width, p.inv_width, p.eps, slots + 3);
        four([&](uint32_t i, auto full) {
            constexpr bool kAll = decltype(full)::value == 4;
            float w[4] = {1.0f, 1.0f, 1.0f, 1.0f}, n[4];
            if (p.pre_w) {
                if (p.w_f32) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) w[e] = kAll || i + e * T < p.width ? load_one(p.pre_w, 1, i + e * T) : 0.0f;
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) w[e] = kAll || i + e * T < p.width ? load_one(p.pre_w, 0, i + e * T) : 0.0f;
                }
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) n[e] = kAll || i + e * T < p.width ? row_mem[i + e * T] * r2 * w[e] : 0.0f;
            if (p.n_f32) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (kAll || i + e * T < p.width) store_one(p.n_out, 1, no + i + e * T, n[e]);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (kAll || i + e * T < p.width) store_one(p.n_out, 0, no + i + e * T, n[e]);
            }
        });
    }
}

constexpr uint32_t kNormMaxWidth = 32768;            // 1,024 threads x 32 elements

}  // namespace m26b
