// C ABI of the dense operators around the routed experts: the MXFP4 linear / gated projections (linear_w4.cuh) and the step
// between two blocks (block_norm.cuh). Included into the library's single translation unit behind m26b_api.cu's helpers.
#pragma once
#include <new>

#include "linear_rules.h"

struct m26b_linear {
    uint8_t *w = nullptr, *sf = nullptr;        // weight image (linear_w4.cuh)
    uint32_t n = 0, k = 0, k_pad = 0;
    bool gated = false;
    int device = 0, sms = 0;
    uint32_t tiles = 0;                         // 128-row tiles of the image (even)
    m26b::LinearShape shape{};                  // the same for the host's rules, with what the device can place
    long long wait_cycles = kWaitCycles;        // bound of the epilogues' wait for their accumulators
    CUtensorMap map_w, map_sf;
};

namespace {

static_assert(linear_widest_pair_tile(true) == LinearPairTile<2>::kTokens && linear_widest_pair_tile(false) == LinearPairTile<1>::kTokens &&
              kChunkK == 128 && kScaleBlockBytes == 512, "linear_rules.h knows the kernels' widest tiles, a chunk and a scale block");
constexpr uint32_t kLinearMaxDim = 1u << 20;
constexpr uint32_t kDenseMaxRows = 0x7fffffffu;

// Asked about in place of the product's kernels, never launched: for a kernel that allocates tensor memory the occupancy calls answer one CTA
// per SM whatever it needs (256 CTAs of 4,096 x 16,384 for one token, two on most SMs: 10.3 us; the 128 that the calls grant: 15.1).
__global__ void linear_room_kernel() {}

// CTAs that run at once in clusters of 1 << log_size (0 if the device cannot place one): GPCs hold whole clusters, and not all have the same SMs.
template <int B_ROWS>
cudaError_t linear_room(int sms, uint32_t (&room)[4]) {
    using T = LinearTile<B_ROWS, 2>;
    const int smem = int(sizeof(LinearSmem<B_ROWS, 2>)) + 1024;
    // the most a CTA may have, whatever is asked: another thread may be between its setting and its asking
    const cudaError_t e = cudaFuncSetAttribute(linear_room_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return e;
    room[0] = uint32_t(sms * T::kCtasPerSm);
    for (uint32_t log_size = 1; log_size < 4; ++log_size) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(room[0] >> log_size << log_size); cfg.blockDim = dim3(T::kThreads); cfg.dynamicSmemBytes = size_t(smem);
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = 1u << log_size; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
        cfg.attrs = &at; cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, linear_room_kernel, &cfg) != cudaSuccess) { clusters = 0; cudaGetLastError(); }
        const uint32_t ctas = uint32_t(clusters) << log_size;
        room[log_size] = ctas < room[0] ? ctas : room[0];
    }
    return cudaSuccess;
}

int linear_new(const uint8_t* const (&w)[2], const uint8_t* const (&s)[2], bool gated, uint32_t n, uint32_t k, m26b_linear** out, char* err,
               size_t errlen) {
    if (!out || !w[0] || !s[0] || (gated && (!w[1] || !s[1])) || !n || n > kLinearMaxDim || !k || k > kLinearMaxDim || k % kBlockK) {
        set_msg(err, errlen, "m26b linear: bad tensors/extents (k a multiple of 32)");
        return 1;
    }
    *out = nullptr;
    m26b_linear* L = new (std::nothrow) m26b_linear;
    if (!L) { set_msg(err, errlen, "m26b linear: out of host memory"); return 2; }
    L->n = n; L->k = k; L->gated = gated;
    L->k_pad = (k + kChunkK - 1) / kChunkK * kChunkK;
    const uint32_t feats = gated ? kTileM : kPairM;                    // output features of two tiles
    L->tiles = (n + feats - 1) / feats * 2;
    const uint64_t rows = uint64_t(L->tiles) * kTileM, chunks = L->k_pad / kChunkK;
    const uint64_t w_bytes = rows * (L->k_pad / 2), sf_bytes = L->tiles * chunks * kScaleBlockBytes;
    auto fail = [&](const char* what, cudaError_t e) {
        set_err(err, errlen, what, e);
        m26b_linear_free(L);
        return 2;
    };
    cudaError_t e = cudaGetDevice(&L->device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&L->sms, cudaDevAttrMultiProcessorCount, L->device);
    if (e != cudaSuccess) return fail("m26b linear device", e);
    L->shape.tiles = L->tiles; L->shape.chunks = uint32_t(chunks); L->shape.sms = uint32_t(L->sms);
    if ((e = linear_room<128>(L->sms, L->shape.room[0])) != cudaSuccess || (e = linear_room<16>(L->sms, L->shape.room[1])) != cudaSuccess)
        return fail("m26b linear occupancy", e);
    if ((e = cudaDeviceSynchronize()) != cudaSuccess) return fail("m26b linear sync", e);      // the source may come from any stream
    void* mem = nullptr;
    if ((e = cudaMalloc(&mem, w_bytes)) != cudaSuccess) return fail("m26b linear weights alloc", e);
    L->w = static_cast<uint8_t*>(mem);
    if ((e = cudaMalloc(&mem, sf_bytes)) != cudaSuccess) return fail("m26b linear scales alloc", e);
    L->sf = static_cast<uint8_t*>(mem);
    const LinearSrc src{{w[0], w[1]}, {s[0], s[1]}};
    linear_prep_payload_kernel<<<L->sms * 8, 256>>>(src, gated, n, k, L->k_pad, rows, L->w);
    linear_prep_scales_kernel<<<L->sms * 8, 256>>>(src, gated, n, k, uint32_t(chunks), sf_bytes, L->sf);
    if ((e = cudaGetLastError()) != cudaSuccess) return fail("m26b linear prepare launch", e);
    if ((e = cudaDeviceSynchronize()) != cudaSuccess) return fail("m26b linear prepare", e);
    if (!make_map(&L->map_w, true, L->w, L->k_pad, rows, L->k_pad / 2, kTileM) || !make_sf_map(&L->map_sf, L->sf, L->tiles * chunks, 1)) {
        set_msg(err, errlen, "m26b linear: cuTensorMapEncodeTiled failed for the weights");
        m26b_linear_free(L);
        return 2;
    }
    *out = L;
    return 0;
}

template <int B_ROWS, int PIECES, bool GATED, bool DIRECT>
cudaError_t launch_linear(const m26b_linear* L, const TokenMaps& mx, const LinearArgs& a, cudaStream_t st) {
    using T = LinearTile<B_ROWS, PIECES>;
    const auto kernel = linear_w4_kernel<B_ROWS, PIECES, GATED, DIRECT>;
    const int smem = int(sizeof(LinearSmem<B_ROWS, PIECES>)) + 1024;
    static std::atomic<uint64_t> opted{0};                             // one flag bit per device of this process
    const uint64_t bit = 1ull << (L->device & 63);
    if (!(opted.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        opted.fetch_or(bit, std::memory_order_relaxed);
    }
    const uint32_t feats = GATED ? 64 : kTileM, tiles = (a.n + feats - 1) / feats, tok_tiles = (a.rows + B_ROWS - 1) / B_ROWS;
    const uint32_t log_split = linear_log_split(L->shape, uint64_t(tiles) * tok_tiles, T::kCtasPerSm, a.chunks);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles << log_split, tok_tiles); cfg.blockDim = dim3(T::kThreads); cfg.dynamicSmemBytes = size_t(smem); cfg.stream = st;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 1u << log_split; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, L->map_w, mx, a, log_split);
}
template <int B_ROWS, bool DIRECT>
cudaError_t launch_linear_tile(const m26b_linear* L, bool bf16, const TokenMaps& mx, const LinearArgs& a, cudaStream_t st) {
    if (L->gated) return bf16 ? launch_linear<B_ROWS, 2, true, DIRECT>(L, mx, a, st) : launch_linear<B_ROWS, 1, true, DIRECT>(L, mx, a, st);
    return bf16 ? launch_linear<B_ROWS, 2, false, DIRECT>(L, mx, a, st) : launch_linear<B_ROWS, 1, false, DIRECT>(L, mx, a, st);
}

// How many CTAs of the pair kernel the device holds at once (an even number, at most one per SM); 0 if it cannot place a pair.
template <int PIECES, bool GATED>
int linear_pair_ctas(const m26b_linear* L) {
    static std::atomic<int> known[64]{};                               // by device of this process: CTAs + 1
    std::atomic<int>& mine = known[L->device & 63];
    int ctas = mine.load(std::memory_order_relaxed);
    if (ctas) return ctas - 1;
    const auto kernel = linear_pair_kernel<PIECES, GATED>;
    const int smem = int(sizeof(LinearPairSmem<PIECES>)) + 1024;
    int clusters = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(unsigned(L->sms & ~1)); cfg.blockDim = dim3(kLpThreads); cfg.dynamicSmemBytes = size_t(smem);
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
        cfg.attrs = &at; cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) clusters = 0;
    }
    cudaGetLastError();
    ctas = 2 * clusters < (L->sms & ~1) ? 2 * clusters : (L->sms & ~1);
    mine.store(ctas + 1, std::memory_order_relaxed);
    return ctas;
}
uint32_t linear_pair_ctas(const m26b_linear* L, bool bf16) {
    if (L->gated) return uint32_t(bf16 ? linear_pair_ctas<2, true>(L) : linear_pair_ctas<1, true>(L));
    return uint32_t(bf16 ? linear_pair_ctas<2, false>(L) : linear_pair_ctas<1, false>(L));
}
template <int PIECES, bool GATED>
cudaError_t launch_linear_pair(const m26b_linear* L, const LinearPairMaps& maps, const LinearArgs& a, uint32_t tile, cudaStream_t st) {
    const uint32_t m_pairs = L->tiles / 2, items = m_pairs * ((a.rows + tile - 1) / tile);
    const uint32_t room = uint32_t(linear_pair_ctas<PIECES, GATED>(L));
    return launch_dependent(linear_pair_kernel<PIECES, GATED>, 2 * items < room ? 2 * items : room, kLpThreads, sizeof(LinearPairSmem<PIECES>) + 1024, st,
                            maps, a, m_pairs, items, tile);
}
cudaError_t launch_stage(void (*kernel)(SplitArgs), dim3 grid, const SplitArgs& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(256); cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// One pass of at most kLinearPassRows tokens.
int linear_pass(const m26b_linear* L, const void* x, bool bf16, const uint8_t* x_scales, uint64_t x_pitch, uint32_t rows, void* y, int y_f32,
                uint64_t y_pitch, uint8_t* ws, uint32_t* fault, cudaStream_t st, char* err, size_t errlen) {
    const uint32_t pieces = bf16 ? 2 : 1, rows_cap = linear_rows_cap(rows);
    const uintptr_t xa = reinterpret_cast<uintptr_t>(x);
    const int vec = bf16 ? (xa % 16 == 0 && x_pitch % 8 == 0) : (xa % 8 == 0 && x_pitch % 8 == 0);
    uint8_t* sf = ws + uint64_t(pieces) * rows_cap * L->k_pad;
    const LinearArgs a{L->sf, sf, rows, rows_cap, L->n, L->k_pad / kChunkK, y, y_f32, y_pitch, fault, x, x_scales, x_pitch, L->k,
                       L->wait_cycles};
    TokenMaps mx{};
    cudaError_t e;
    const uint32_t pair_tile = rows <= 128 ? 0 : linear_pair_tile(L->shape, linear_pair_ctas(L, bf16), bf16, rows), tile = pair_tile ? pair_tile : rows <= 64 ? 64u : 128u;
    if (vec && !pair_tile && linear_direct(L->shape, bf16, rows)) {
        if (rows <= 16) e = launch_linear_tile<16, true>(L, bf16, mx, a, st);
        else if (rows <= 32) e = launch_linear_tile<32, true>(L, bf16, mx, a, st);
        else if (rows <= 64) e = launch_linear_tile<64, true>(L, bf16, mx, a, st);
        else e = launch_linear_tile<128, true>(L, bf16, mx, a, st);
    } else {
        const SplitArgs sp{x, x_scales, x_pitch, rows, L->k, L->k_pad, rows_cap, tile, rows <= 64 ? 1u : 0u, ws, sf};
        // quantised rows on 16-byte boundaries are loaded from where they are
        const bool in_place = !bf16 && xa % 16 == 0 && x_pitch % 16 == 0;
        if (in_place) e = launch_stage(linear_scales_kernel, dim3((sp.k_pad / kChunkK + 31) / 32, (rows + 7) / 8), sp, st);
        else {
            const dim3 grid((sp.k_pad / kChunkK + 7) / 8, (rows + 7) / 8);
            if (bf16) e = launch_stage(vec ? linear_split_kernel<2, true> : linear_split_kernel<2, false>, grid, sp, st);
            else e = launch_stage(vec ? linear_split_kernel<1, true> : linear_split_kernel<1, false>, grid, sp, st);
        }
        if (e != cudaSuccess) { cudaGetLastError(); set_err(err, errlen, "m26b linear stage launch", e); return 2; }
        const uint64_t map_rows = in_place ? rows : uint64_t(pieces) * rows_cap, map_cols = in_place ? L->k : L->k_pad, map_pitch = in_place ? x_pitch : L->k_pad;
        void* map_base = in_place ? const_cast<void*>(x) : ws;
        const auto boxes = [&](CUtensorMap* to, int count) {            // the boxes a token tile of this request can use
            for (int i = 0; i < count; ++i)
                if ((128u >> i) <= rows_cap && !make_map(&to[i], false, map_base, map_cols, map_rows, map_pitch, 128u >> i)) return false;
            return true;
        };
        bool maps_ok;
        if (pair_tile) {
            LinearPairMaps pm{};
            pm.w = L->map_w; pm.sfa = L->map_sf;
            const uint32_t blocks = (tile > 128 ? 2 : 1) * pieces;
            maps_ok = boxes(pm.tok, 5) && make_sf_map(&pm.sfb, sf, linear_scale_blocks(rows, tile, pieces) * a.chunks, blocks);
            if (maps_ok) {
                if (L->gated) e = bf16 ? launch_linear_pair<2, true>(L, pm, a, tile, st) : launch_linear_pair<1, true>(L, pm, a, tile, st);
                else e = bf16 ? launch_linear_pair<2, false>(L, pm, a, tile, st) : launch_linear_pair<1, false>(L, pm, a, tile, st);
            }
        } else {
            maps_ok = boxes(mx.box, 4);
            if (maps_ok) e = rows <= 64 ? launch_linear_tile<64, false>(L, bf16, mx, a, st) : launch_linear_tile<128, false>(L, bf16, mx, a, st);
        }
        if (!maps_ok) { set_msg(err, errlen, "m26b linear: cuTensorMapEncodeTiled failed for the activations"); return 2; }
    }
    if (e != cudaSuccess) { cudaGetLastError(); set_err(err, errlen, "m26b linear launch", e); return 2; }
    return 0;
}

// SMs of a device, 0 if it cannot be asked.
uint32_t device_sms(int dev) {
    static std::atomic<uint32_t> known[64]{};                          // by device of this process
    uint32_t sms = known[dev & 63].load(std::memory_order_relaxed);
    if (!sms) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { cudaGetLastError(); return 0; }
        known[dev & 63].store(sms = uint32_t(n), std::memory_order_relaxed);
    }
    return sms;
}
// Rows are strided over by as many CTAs as the GPU holds at once.
template <int VEC, int PER, int THREADS, bool Y32, bool H32, bool GATE_ELEM>
cudaError_t launch_norm_kernel(const NormArgs& a, int dev, cudaStream_t st) {
    const auto kernel = block_norm_kernel<VEC, PER, THREADS, Y32, H32, GATE_ELEM>;
    constexpr uint32_t block = THREADS == 32 ? 128 : THREADS;
    static std::atomic<uint32_t> known[64]{};                          // CTAs the device holds, by device of this process
    uint32_t room = known[dev & 63].load(std::memory_order_relaxed);
    if (!room) {
        int per_sm = 0;
        const uint32_t sms = device_sms(dev);
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, int(block), 0);
        if (e != cudaSuccess || per_sm < 1 || !sms) return e != cudaSuccess ? e : cudaErrorLaunchOutOfResources;
        room = sms * uint32_t(per_sm);
        known[dev & 63].store(room, std::memory_order_relaxed);
    }
    const uint32_t need = THREADS == 32 ? (a.rows + 3) / 4 : a.rows;
    return launch_dependent(kernel, need < room ? need : room, block, 0, st, a);
}
template <int VEC, int PER, int THREADS>
cudaError_t launch_norm(const NormArgs& a, int dev, cudaStream_t st) {
    const auto typed = [&](auto y32, auto h32) {
        if (a.gate_kind == kGateElement) return launch_norm_kernel<VEC, PER, THREADS, y32.value, h32.value, true>(a, dev, st);
        return launch_norm_kernel<VEC, PER, THREADS, y32.value, h32.value, false>(a, dev, st);
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    if (a.y_f32) return a.h_f32 ? typed(yes, yes) : typed(yes, no);
    return a.h_f32 ? typed(no, yes) : typed(no, no);
}
// Threads and vectors per thread by width: a row's CTA is as small as its registers allow (8,192 x 4,096: 62 us with two vectors of
// eight in each of 256 threads, 87 with one in 512, 72 with four in 128), since what a row costs beyond its bytes is two
// reductions over its threads. Wider rows than 8,192 do not fit the registers of a CTA and take block_norm_any_kernel.
cudaError_t launch_norm_vec8(const NormArgs& a, int dev, cudaStream_t st) {
    if (a.width <= 512) return launch_norm<8, 2, 32>(a, dev, st);
    if (a.width <= 1024) return launch_norm<8, 2, 64>(a, dev, st);
    if (a.width <= 2048) return launch_norm<8, 2, 128>(a, dev, st);
    if (a.width <= 4096) return launch_norm<8, 2, 256>(a, dev, st);
    return launch_norm<8, 2, 512>(a, dev, st);
}
cudaError_t launch_norm_vec4(const NormArgs& a, int dev, cudaStream_t st) {
    if (a.width <= 1024) return launch_norm<4, 4, 64>(a, dev, st);
    if (a.width <= 4096) return launch_norm<4, 4, 256>(a, dev, st);
    return launch_norm<4, 4, 512>(a, dev, st);
}
template <uint32_t T, bool Y32, bool H32>
cudaError_t launch_norm_any(const NormArgs& a, int dev, cudaStream_t st) {
    const auto kernel = block_norm_any_kernel<T, Y32, H32>;
    const size_t smem = size_t(a.width) * 4;
    static std::atomic<uint64_t> opted{0};                             // one flag bit per device of this process
    const uint64_t bit = 1ull << (dev & 63);
    if (!(opted.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kNormMaxWidth) * 4);
        if (e != cudaSuccess) return e;
        opted.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch_dependent(kernel, a.rows, T, smem, st, a);
}
template <bool Y32, bool H32>
cudaError_t launch_norm_any_width(const NormArgs& a, int dev, cudaStream_t st) {
    // more rows than large CTAs fit the device (two per SM): CTAs so small that eight of them share an SM (8,192 x 4,095: 101 us, 178 with
    // 1,024 threads); fewer: the threads of one SM on one row (1 x 4,095: 4.4 us, 7.0 with 256)
    if (a.width <= 512) return launch_norm_any<64, Y32, H32>(a, dev, st);
    if (a.width <= 1024 || (a.width <= 8192 && a.rows > 2 * device_sms(dev))) return launch_norm_any<256, Y32, H32>(a, dev, st);
    return launch_norm_any<1024, Y32, H32>(a, dev, st);
}

}  // namespace

extern "C" {

int m26b_linear_new(const uint8_t* w, const uint8_t* s, uint32_t n, uint32_t k, m26b_linear** out, char* err, size_t errlen) {
    const uint8_t *ws[2] = {w, nullptr}, *ss[2] = {s, nullptr};
    return linear_new(ws, ss, false, n, k, out, err, errlen);
}
int m26b_linear_new_gated(const uint8_t* gate_w, const uint8_t* gate_s, const uint8_t* up_w, const uint8_t* up_s, uint32_t n, uint32_t k,
                          m26b_linear** out, char* err, size_t errlen) {
    const uint8_t *ws[2] = {gate_w, up_w}, *ss[2] = {gate_s, up_s};
    return linear_new(ws, ss, true, n, k, out, err, errlen);
}
void m26b_linear_free(m26b_linear* l) {
    if (!l) return;
    if (l->w) cudaFree(l->w);
    if (l->sf) cudaFree(l->sf);
    delete l;
}
int m26b_linear_set_wait_us(m26b_linear* l, uint32_t us) {
    if (!l || !us) return 1;
    int khz = 0;                                // nominal SM clock; the call takes half a millisecond, so not in every linear_new
    if (cudaDeviceGetAttribute(&khz, cudaDevAttrClockRate, l->device) != cudaSuccess || khz <= 0) { cudaGetLastError(); khz = 1965000; }
    l->wait_cycles = (long long)us * khz / 1000;
    return 0;
}
uint64_t m26b_linear_workspace_bytes(const m26b_linear* l, uint32_t rows) {
    return l ? linear_workspace(l->k_pad, rows) : 0;
}
int m26b_linear_dev(const m26b_linear* l, const m26b_linear_args* args, void* stream, char* err, size_t errlen) {
    if (!l || !args || !(args->x_dtype == 0 || args->x_dtype == 2) || args->y_dtype < 0 || args->y_dtype > 1 || args->reserved) {
        set_msg(err, errlen, "m26b linear: bad handle/dtype (x 0 BF16 or 2 E4M3, y 0 BF16 or 1 FP32)");
        return 1;
    }
    const m26b_linear_args& in = *args;
    const uint32_t rows = in.rows;
    if (!rows) return 0;
    const bool bf16 = in.x_dtype == 0;
    const uint64_t x_pitch = in.x_pitch ? in.x_pitch : l->k, y_pitch = in.y_pitch ? in.y_pitch : l->n;
    if (rows > kDenseMaxRows || !in.x || !in.y || !in.fault_dev || (!bf16 && !in.x_scales) || x_pitch < l->k || y_pitch < l->n) {
        set_msg(err, errlen, "m26b linear: bad pointers/pitch/rows");
        return 1;
    }
    if ((bf16 && reinterpret_cast<uintptr_t>(in.x) % 2) || reinterpret_cast<uintptr_t>(in.y) % (in.y_dtype ? 4 : 2) ||
        reinterpret_cast<uintptr_t>(in.fault_dev) % 4) {
        set_msg(err, errlen, "m26b linear: x, y or the fault word is not aligned to its element size");
        return 1;
    }
    if (!in.workspace || reinterpret_cast<uintptr_t>(in.workspace) % 128 || in.workspace_bytes < m26b_linear_workspace_bytes(l, rows)) {
        set_msg(err, errlen, "m26b linear: workspace too small or not 128-byte aligned (m26b_linear_workspace_bytes)");
        return 1;
    }
    int dev = -1;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) { set_err(err, errlen, "m26b linear device", e); return 2; }
    if (dev != l->device) { set_msg(err, errlen, "m26b linear: the handle belongs to another device"); return 1; }
    const uint64_t x_row = x_pitch * (bf16 ? 2 : 1), y_row = y_pitch * (in.y_dtype ? 4 : 2);
    for (uint32_t r0 = 0; r0 < rows; r0 += kLinearPassRows) {
        const uint32_t m = rows - r0 < kLinearPassRows ? rows - r0 : kLinearPassRows;
        const int rc = linear_pass(l, static_cast<const uint8_t*>(in.x) + r0 * x_row, bf16, bf16 ? nullptr : in.x_scales + uint64_t(r0) * (l->k / kBlockK),
                                   x_pitch, m, static_cast<uint8_t*>(in.y) + r0 * y_row, in.y_dtype, y_pitch, static_cast<uint8_t*>(in.workspace),
                                   in.fault_dev, static_cast<cudaStream_t>(stream), err, errlen);
        if (rc) return rc;
    }
    return 0;
}

int m26b_block_norm_dev(const m26b_block_norm_args* args, void* stream, char* err, size_t errlen) {
    if (!args) { set_msg(err, errlen, "m26b block norm: bad arguments"); return 1; }
    const m26b_block_norm_args& in = *args;
    const int n_planes = in.n_planes, y_dtype = in.y_dtype, h_dtype = in.h_dtype, n_dtype = in.n_dtype, w_dtype = in.w_dtype, gate_kind = in.gate_kind;
    const uint32_t rows = in.rows, width = in.width;
    const auto bad = [](int t) { return t < 0 || t > 1; };
    if (n_planes < 0 || n_planes > 8 || bad(y_dtype) || bad(h_dtype) || bad(w_dtype) || bad(n_dtype) || gate_kind < 0 || gate_kind > 3 || in.reserved ||
        (gate_kind != 0) != (in.gate != nullptr) || (!n_planes && (in.post_w || in.gate || !in.residual)) || (!in.h_out && !in.n_out) ||
        (!in.n_out && in.pre_w) || !width || width > kNormMaxWidth || rows > kDenseMaxRows) {
        set_msg(err, errlen, "m26b block norm: bad arguments");
        return 1;
    }
    // a square that FP32 holds in part or not at all is off by 2^-150 at most: nothing beside a normal eps, but not beside a subnormal one
    if (!(in.eps >= 0x1p-126f) || in.eps > 3.0e38f) { set_msg(err, errlen, "m26b block norm: eps must be positive, at least 2^-126"); return 1; }
    const uint64_t y_pitch = in.y_pitch ? in.y_pitch : width, h_pitch = in.h_pitch ? in.h_pitch : width, n_pitch = in.n_pitch ? in.n_pitch : width;
    if (y_pitch < width || h_pitch < width || n_pitch < width) { set_msg(err, errlen, "m26b block norm: a pitch is below the width"); return 1; }
    NormArgs a{};
    uintptr_t vec8 = 0, vec4 = 0, elem = 0;           // address bits that keep vectors of 8 / of 4 / single elements from being aligned
    const auto see = [&](const void* p, int f32) {
        const uintptr_t v = reinterpret_cast<uintptr_t>(p);
        vec8 |= v & 15; vec4 |= v & (f32 ? 15 : 7); elem |= v & (f32 ? 3 : 1);
    };
    for (int r = 0; r < n_planes; ++r) {
        if (!in.planes[r]) { set_msg(err, errlen, "m26b block norm: bad arguments"); return 1; }
        a.y[r] = in.planes[r];
        see(in.planes[r], y_dtype);
    }
    a.planes = n_planes;
    a.y_f32 = y_dtype; a.h_f32 = h_dtype; a.n_f32 = n_dtype; a.w_f32 = w_dtype;
    a.y_pitch = y_pitch; a.h_pitch = h_pitch; a.n_pitch = n_pitch;
    a.post_w = in.post_w; a.gate = in.gate; a.residual = in.residual; a.pre_w = in.pre_w;
    a.gate_kind = gate_kind;
    a.y_scale = n_planes ? in.y_scale : 1.0f; a.residual_scale = in.residual ? in.residual_scale : 0.0f; a.eps = in.eps;
    a.inv_width = 1.0f / float(width);
    a.rows = rows; a.width = width; a.h_out = in.h_out; a.n_out = in.n_out;
    see(in.post_w, w_dtype); see(in.pre_w, w_dtype); see(in.residual, h_dtype); see(in.h_out, h_dtype); see(in.n_out, n_dtype);
    if (gate_kind == kGateToken) elem |= reinterpret_cast<uintptr_t>(in.gate) & 3;
    else see(in.gate, gate_kind == kGateChannel ? w_dtype : y_dtype);
    if (elem) { set_msg(err, errlen, "m26b block norm: a pointer is not aligned to its element size"); return 1; }
    if (!rows) return 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint64_t pitches = (n_planes ? y_pitch : 0) | (in.residual || in.h_out ? h_pitch : 0) | (in.n_out ? n_pitch : 0);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) { set_err(err, errlen, "m26b block norm device", e); return 2; }
    if (!vec8 && (width | pitches) % 8 == 0 && width <= 8192) e = launch_norm_vec8(a, dev, st);
    else if (!vec4 && pitches % 4 == 0 && width <= 8192) e = launch_norm_vec4(a, dev, st);
    else if (y_dtype) e = h_dtype ? launch_norm_any_width<true, true>(a, dev, st) : launch_norm_any_width<true, false>(a, dev, st);
    else e = h_dtype ? launch_norm_any_width<false, true>(a, dev, st) : launch_norm_any_width<false, false>(a, dev, st);
    if (e != cudaSuccess) { cudaGetLastError(); set_err(err, errlen, "m26b block norm launch", e); return 2; }
    return 0;
}

}  // extern "C"
