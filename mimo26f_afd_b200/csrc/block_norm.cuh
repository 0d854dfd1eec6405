// The step between two blocks of a decoder, one pass over each row:
//     u = y_0 + y_1 + ... (rank order)          the block's output, one BF16 plane per rank or one FP32 plane
//     u = u / sqrt(mean(u^2) + eps) * post_w    norm after the block (optional)
//     h = residual_scale * residual + y_scale * gate * u
//     n = h / sqrt(mean(h^2) + eps) * pre_w     norm before the next block (optional)
// The reference runs it as three launches on the coordinator (rank sum, h += f, rmsnorm:
// crates/mimo26-coordinator/kernels/glue.cu:55-59, 200-213); the operands of a row are read once here and the row stays
// in registers between the two reductions. Everything is FP32 from the loads to the single rounding of each output.
//
// What bounds it: HBM traffic (planes + residual in, h and n out); about twelve operations per element.
// Layout: a row belongs to a warp (narrow rows) or a CTA; a thread owns PER vectors of VEC elements, a row's worth apart, so
// that every access of a warp is one contiguous run.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

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
    float y_scale, residual_scale, eps, inv_width;      // y_scale 0 without planes, residual_scale 0 without a residual
    uint32_t rows, width;
    void *h_out, *n_out;
};

// VEC consecutive elements starting at element `i`; VEC = 8 needs 16-byte alignment.
template <int VEC>
__device__ __forceinline__ void load_elems(const void* base, int f32, uint64_t i, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = f32 ? static_cast<const float*>(base)[i] : __uint_as_float(uint32_t(static_cast<const uint16_t*>(base)[i]) << 16);
    } else if (f32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
        const float4 a = p[0], b = p[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
    }
}
// Two floats as BF16 (nearest even, NaN kept), the first in the low half.
__device__ __forceinline__ uint32_t bf16x2_rn(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int VEC>
__device__ __forceinline__ void store_elems(void* base, int f32, uint64_t i, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        if (f32) static_cast<float*>(base)[i] = v[0];
        else static_cast<uint16_t*>(base)[i] = uint16_t(bf16x2_rn(v[0], 0.0f));
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

// VEC elements as they lie in memory: loads are issued for a whole row before anything waits for one of them.
template <int VEC, bool F32>
struct RawVec {
    uint32_t w[VEC == 1 ? 1 : VEC * (F32 ? 4 : 2) / 4];
    __device__ __forceinline__ void load(const void* base, uint64_t i) {
        if constexpr (VEC == 1) {
            if constexpr (F32) w[0] = static_cast<const uint32_t*>(base)[i];
            else w[0] = static_cast<const uint16_t*>(base)[i];
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

// A row belongs to a warp (MAX_THREADS 128: four rows per CTA) or to a CTA; both stride over the rows by the grid, and the
// next row's operands are requested before this row's reductions are waited for. Y32 / H32: FP32 planes / residual stream.
template <int VEC, int PER, int MAX_THREADS, bool Y32, bool H32>
__global__ void __launch_bounds__(MAX_THREADS) block_norm_kernel(const NormArgs p) {
    constexpr bool BLOCK = MAX_THREADS > 128;
    __shared__ float slots_all[2][6][32];
    const uint32_t threads = BLOCK ? blockDim.x : 32u;
    const uint32_t t = BLOCK ? threadIdx.x : threadIdx.x & 31u;
    const uint32_t rows_at_once = BLOCK ? gridDim.x : gridDim.x * (blockDim.x >> 5);
    uint32_t row = BLOCK ? blockIdx.x : blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    RawVec<VEC, Y32> ry[PER], rg[PER];
    RawVec<VEC, H32> rh[PER];
    const bool has_y = p.planes > 0, has_h = p.residual != nullptr, gate_elem = p.gate_kind == kGateElement;
    const auto request = [&](uint32_t r) {
        const uint64_t yo = uint64_t(r) * p.y_pitch, ho = uint64_t(r) * p.h_pitch;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = (t + j * threads) * VEC;
            if (i < p.width) {
                if (has_y) ry[j].load(p.y[0], yo + i);
                if (has_h) rh[j].load(p.residual, ho + i);
                if (gate_elem) rg[j].load(p.gate, yo + i);
            }
        }
    };
#pragma unroll
    for (int j = 0; j < PER; ++j) { ry[j].zero(); rh[j].zero(); rg[j].zero(); }
    grid_dep_wait();                                 // the block's output comes from the stream's earlier kernels
    grid_dep_launch();
    if (row < p.rows) request(row);
    for (uint32_t turn = 0; row < p.rows; row += rows_at_once, ++turn) {
        float (*slots)[32] = slots_all[turn & 1];    // the other set may still be read by slower warps of the row before
        const uint64_t yo = uint64_t(row) * p.y_pitch, ho = uint64_t(row) * p.h_pitch, no = uint64_t(row) * p.n_pitch;
        float u[PER * VEC], h[PER * VEC];
        RawVec<VEC, Y32> cg[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            cg[j] = rg[j];
#pragma unroll
            for (int e = 0; e < VEC; ++e) { u[j * VEC + e] = ry[j].get(e); h[j * VEC + e] = rh[j].get(e); }
        }
        if (p.planes > 1) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const uint32_t i = (t + j * threads) * VEC;
                if (i >= p.width) continue;
                RawVec<VEC, Y32> more[7];
#pragma unroll
                for (int q = 0; q < 7; ++q) {
                    more[q].zero();
                    if (q + 1 < p.planes) more[q].load(p.y[q + 1], yo + i);
                }
#pragma unroll
                for (int q = 0; q < 7; ++q) {
                    if (q + 1 >= p.planes) break;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) u[j * VEC + e] += more[q].get(e);
                }
            }
        }
        if (rows_at_once < p.rows - row) request(row + rows_at_once);
        float r1 = p.y_scale;                          // every factor of u that the row shares
        if (p.gate_kind == kGateToken) r1 *= static_cast<const float*>(p.gate)[row];
        if (p.post_w) r1 *= row_rrms<PER * VEC, BLOCK>(u, p.inv_width, p.eps, slots);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = (t + j * threads) * VEC;
            if (i >= p.width) continue;
            float a[VEC], w[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = u[j * VEC + e] * r1;
            if (p.post_w) {
                load_elems<VEC>(p.post_w, p.w_f32, i, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= w[e];
            }
            if (gate_elem) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= cg[j].get(e);
            } else if (p.gate_kind == kGateChannel) {
                load_elems<VEC>(p.gate, p.w_f32, i, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= w[e];
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = fmaf(h[j * VEC + e], p.residual_scale, a[e]);
            if (p.h_out) store_elems<VEC>(p.h_out, H32, ho + i, a);
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[j * VEC + e] = a[e];
        }
        if (!p.n_out) continue;
        const float r2 = row_rrms<PER * VEC, BLOCK>(h, p.inv_width, p.eps, slots + 3);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = (t + j * threads) * VEC;
            if (i >= p.width) continue;
            float a[VEC], w[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = h[j * VEC + e] * r2;
            if (p.pre_w) {
                load_elems<VEC>(p.pre_w, p.w_f32, i, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) a[e] *= w[e];
            }
            store_elems<VEC>(p.n_out, p.n_f32, no + i, a);
        }
    }
}

constexpr uint32_t kNormMaxWidth = 32768;            // 1,024 threads x 32 elements

}  // namespace m26b
