// f8blk_plan.cuh - which kernel a product of block-scaled e4m3 operands takes.  Host code without CUDA calls.
//
// The estimates, us, were fitted to measured times of 100 random shapes (in 512 ... 17408, out 512 ... 17408, 1 ... 1500 tokens; gemm and gated
// front) under every plan, cold weights.  The plan they pick takes 1.6 % longer than the best of the plans on average, 25 % at worst (3.3
// against 4.1 us).  What they weigh:
//   split   a CTA does its part of K alone and meets its cluster.  One plane: 0.3 or 0.4 us a block of K, 0.2 more beside another CTA, and 1.7 or
//           2.2 us and 25 ns a token for the meeting; where one CTA takes all of K, half of those 25 ns for the stores.  Gated: 0.5 or 1.0 us a block
//           of both planes, 0.35 more beside another CTA, and 74 or 54 ns a token for the meeting, which is there with one CTA too.  Wins where a
//           call has few tiles: 380 tokens, 13760 x 576 gated 25.9 us, wide 52.0
//   wide    0.26 - 0.65 us a block of K and round of tiles.  Wins from the number of tiles on that fills the SMs: 648 tokens, 5888 x 2816 gated
//           27.3 us, split 60.3; 128 channels a tile rather than 256 where those leave SMs empty: 200 tokens, 5120 x 5120 15.2 and 22.2
#pragma once
#include <stdint.h>

namespace f8blk {

struct Plan {
    uint32_t kernel;   // 1 split, 2 wide
    uint32_t cols;     // split: tokens of a tile (32, 64); wide: channels of a tile (128, 256; gated: 256, gate's and up's)
    uint32_t split;    // split: CTAs that share a tile
};

static inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1u) / b; }

// The largest split whose clusters are all resident at once, of at least two blocks of K each.  resident[s]: clusters of s CTAs by the driver,
// which counts one CTA per SM for a kernel that allocates tensor memory; two run.
static inline uint32_t largest_split(uint64_t tiles, uint32_t blocks, const uint32_t* resident, uint32_t most) {
    uint32_t split = blocks / 2u < most ? blocks / 2u : most;
    while (split > 1u && tiles > 2u * (uint64_t)resident[split]) --split;
    return split ? split : 1u;
}

static inline double split_us(int planes, uint32_t tok, uint64_t tiles, uint32_t blocks, uint32_t cols, uint32_t split, uint32_t sms) {
    //                                   base  block  block beside another CTA  meeting  a token of it
    static constexpr double kFit[2][2][5] = {{{1.44, 0.30, 0.20, 1.67, 0.027}, {1.32, 0.42, 0.19, 2.15, 0.023}},
                                             {{3.19, 0.51, 0.37, 0.0, 0.074}, {4.45, 1.01, 0.33, 0.0, 0.054}}};
    const double* f = kFit[planes - 1][cols == 32u ? 0 : 1];
    const uint64_t ctas = tiles * split, rounds = ceil_div(ctas, 2u * (uint64_t)sms);
    double beside = ((double)ctas / (double)rounds - sms) / sms;
    beside = beside < 0.0 ? 0.0 : beside > 1.0 ? 1.0 : beside;
    const double meet = split > 1u || planes == 2 ? f[3] + f[4] * tok : 0.5 * f[4] * tok;
    return f[0] + (double)rounds * ((double)ceil_div(blocks, split) * (f[1] + f[2] * beside) + meet);
}

static inline double wide_us(int planes, uint64_t tiles, uint32_t blocks, uint32_t cols, uint32_t sms) {
    //                                base  block  block with all SMs at work  round
    static constexpr double kFit[3][4] = {{2.16, 0.26, 0.15, 0.0}, {2.60, 0.42, 0.23, 0.2}, {4.28, 0.43, 0.17, 0.0}};
    const double* f = kFit[planes == 2 ? 2 : cols == 128u ? 0 : 1];
    const double rounds = (double)ceil_div(tiles, sms), fill = tiles < sms ? (double)tiles / sms : 1.0;
    return f[0] + rounds * (blocks * (f[1] + f[2] * fill) + f[3]);
}

// resident[c]: of the split kernel with 32 << c tokens a tile
static inline Plan choose(int planes, uint32_t in_dim, uint32_t out_dim, uint32_t batch, const uint32_t* const resident[2], uint32_t most,
                          uint32_t sms) {
    const uint32_t blocks = (uint32_t)ceil_div(in_dim, 128u);
    const uint64_t tiles_n = ceil_div(out_dim, 128u), tiles_m = ceil_div(batch, 128u);
    Plan best{};
    double us = 0.0;
    auto offer = [&](uint32_t kernel, uint32_t cols, uint32_t split, double t) {
        if (best.kernel == 0u || t < us) {
            best = Plan{kernel, cols, split};
            us = t;
        }
    };
    for (uint32_t c = 0; c < 2u; ++c) {
        const uint32_t cols = 32u << c, tok = batch < cols ? batch : cols;
        const uint64_t tiles = ceil_div(batch, cols) * tiles_n;
        const uint32_t most_here = largest_split(tiles, blocks, resident[c], most);
        offer(1u, cols, most_here, split_us(planes, tok, tiles, blocks, cols, most_here, sms));
        if (most_here > 1u) offer(1u, cols, 1u, split_us(planes, tok, tiles, blocks, cols, 1u, sms));
        if (batch <= 32u) break;      // 64 columns would be half empty
    }
    if (planes == 1) offer(2u, 128u, 1u, wide_us(planes, tiles_m * tiles_n, blocks, 128u, sms));
    offer(2u, 256u, 1u, wide_us(planes, tiles_m * (planes == 2 ? tiles_n : ceil_div(out_dim, 256u)), blocks, 256u, sms));
    return best;
}

}  // namespace f8blk
