// Sizes and choices of the dense products on the host: what a request's workspace holds, which kernel runs it, in how many parts. Plain
// C++ without CUDA, so that the rules can be checked over their whole range.
#pragma once
#include <cstdint>

namespace m26b {

constexpr uint32_t kLinearPassRows = 8192;      // tokens per pass: bounds the workspace at 2 x 8192 x k bytes
constexpr uint32_t kLinearMinPairTile = 64;     // token tiles of the CTA-pair kernel: multiples of 16 from here
constexpr uint32_t linear_widest_pair_tile(bool bf16) { return bf16 ? 224 : 256; }      // two accumulator sets (two pieces), or one

// What the rules know of a handle and its device.
struct LinearShape {
    uint32_t tiles, chunks;     // 128-row tiles of the weight image, 128-wide chunks of K
    uint32_t sms;
    uint32_t room[2][4];        // [CTAs per SM - 1][log2 of the cluster size]: CTAs that run at once, as the device says
};

inline uint32_t linear_rows_cap(uint32_t rows) { return ((rows < kLinearPassRows ? rows : kLinearPassRows) + 15) & ~15u; }

// Scale blocks (512 bytes) per chunk that a pass of `rows` tokens stages with a token tile: one per 128-token run of a tile and piece, whole tiles;
// up to 64 tokens both pieces share one block.
inline uint64_t linear_scale_blocks(uint32_t rows, uint32_t tile, uint32_t pieces) {
    if (rows <= 64) return 1;
    return uint64_t((rows + tile - 1) / tile) * (tile > 128 ? 2 : 1) * pieces;
}
// The workspace of a request: two pieces of codes, and the scale blocks of whichever token tile is chosen. Tiles of up to 128 tokens need the
// most where they are narrowest (64), wider ones at 144.
inline uint64_t linear_workspace(uint32_t k_pad, uint32_t rows) {
    const uint64_t cap = linear_rows_cap(rows);
    if (!cap) return 0;
    const uint64_t narrow = (cap + 63) / 64, wide = (cap + 143) / 144 * 2;
    return 2 * (cap * k_pad + (narrow > wide ? narrow : wide) * (k_pad / 128) * 512);
}

// log2 of the CTAs that share a weight tile's K (a cluster): doubled while the clusters still run at once and each CTA keeps at least
// two chunks. A GPC holds whole clusters only, so that fewer of them run at once than SMs over cluster size (of the 148 SMs here 33 clusters of
// four and fifteen of eight with one CTA per SM, 71 and 33 with two), and what is left would run as a second round (100 tokens, 2,048 x
// 2,048, sixteen clusters of eight: 15.2 us, of four: 8.3; 16 tokens, 4,224 x 16,384: 11.5 and 16.6). Powers of two: the divisions that
// other sizes need cost 0.3 us, more than they gain.
inline uint32_t linear_log_split(const LinearShape& L, uint64_t ctas, uint32_t per_sm, uint32_t chunks) {
    uint32_t log_split = 0;
    while (log_split < 3 && (ctas << (log_split + 1)) <= L.room[per_sm - 1][log_split + 1] && chunks >= 4u << log_split) ++log_split;
    return log_split;
}
// Whether a request that single CTAs run converts its activations (rows on vector boundaries) inside the product's kernel. Up to 32 tokens
// (64 that arrive quantised) that hides behind the weights; beyond, it pays while a CTA has few chunks, since every weight tile
// repeats it. Measured, inside / staged: 4,096 x 4,096 BF16 32 tokens 8.2 / 9.6 us, 64 10.9 / 8.7, E4M3 64 7.5 / 8.0, 128 11.3 /
// 10.3; 1,000 x 1,024 (two chunks per CTA) BF16 40 tokens 5.2 / 5.6, 128 8.6 / 8.5, each with one launch less.
inline bool linear_direct(const LinearShape& L, bool bf16, uint32_t rows) {
    if (rows <= (bf16 ? 32u : 64u)) return true;
    const uint64_t ctas = uint64_t(L.tiles) * ((rows + 127) / 128);
    const uint32_t per_cta = L.chunks >> linear_log_split(L, ctas, 1, L.chunks);
    return ctas <= L.sms && per_cta * (rows < 128 ? rows : 128) <= (bf16 ? 256u : 512u);
}
// Token tile of the CTA-pair kernel (`ctas`: how many of its CTAs run at once) for a request, or 0 if single CTAs (which can split K)
// finish it sooner, by cycles: rounds of items over the GPU x cycles per item. A 128-wide chunk costs a pair 4 x pieces MMAs, each the
// slower of its math (tile / 2 cycles) and of shared memory at 128 B/clk (weight rows 32 cycles, token rows tile / 8, its share of
// filling the stage); a single CTA of 128 tokens 768 (two pieces) or 512 cycles, shared memory again. The constants are what start, end
// and hand-over of an item cost. A tile narrower than the widest has to win by a tenth: it is more work in all, and the GPU is at
// its power limit (2,048 E4M3 tokens with tiles of 240, 2 % fewer cycles by this count, take 35.5 us, of 256 34.3). Measured (4,096 x
// 4,096, the best pairs / single CTAs): 512 tokens 22.7 / 20.2 us, 768 27.7 / 35.1, 1,024 39.2 / 40.9, 2,048 69.6 / 78.2; E4M3 512 15.8 /
// 12.6, 1,024 19.0 / 25.3.
inline uint32_t linear_pair_tile(const LinearShape& L, uint32_t ctas, bool bf16, uint32_t rows) {
    if (rows <= 128 || ctas < 2) return 0;
    const uint64_t pairs = ctas / 2, m_pairs = L.tiles / 2, pieces = bf16 ? 2 : 1;
    const auto pair_cost = [&](uint32_t tile) {
        const uint64_t rounds = (m_pairs * ((rows + tile - 1) / tile) + pairs - 1) / pairs;
        const uint64_t math = tile / 2, feed = 32 + tile / 8 + (128 + pieces * tile / 2) / (4 * pieces);
        return rounds * (L.chunks * 4 * pieces * (math > feed ? math : feed) + 2000) + 10000;
    };
    const uint32_t widest = linear_widest_pair_tile(bf16);
    uint32_t best = widest;
    uint64_t cost = pair_cost(widest) * 9 / 10;
    for (uint32_t tile = widest - 16; tile >= kLinearMinPairTile; tile -= 16)
        if (pair_cost(tile) < cost) { best = tile; cost = pair_cost(tile); }
    const uint64_t single = uint64_t(L.tiles) * ((rows + 127) / 128), sms = L.sms;
    const uint32_t log_split = linear_log_split(L, single, 1, L.chunks);
    const uint64_t single_cost = ((single << log_split) + sms - 1) / sms * ((L.chunks >> log_split) * (bf16 ? 768 : 512) + 4000);
    return pair_cost(best) < single_cost ? best : 0;
}

}  // namespace m26b
