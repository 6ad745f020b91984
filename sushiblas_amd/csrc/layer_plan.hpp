// layer_plan.hpp -- which kernels the few-token layer (mx4_linear.hip) and the mixture of experts
// (mx4_moe.hip) run: plain arithmetic on their sizes, so that a host program can ask too.
//
// `pieces`: the bf16 pieces that a token's value has (mx4_rows.hpp): 1 of bf16 and MXFP8, 2 of fp16, 3 of fp32.
#pragma once

#include <stdint.h>

namespace sbx {

struct Mx4LinearPlan {
    enum Form {
        Rows,     // linear_kernel
        Tall,     // linear_tall_kernel
        FewTerms  // few_terms_kernel
    } form;
    // of linear_kernel, its template's arguments
    int tokens, tiles, blocks, waves, ahead;
};

inline Mx4LinearPlan mx4_linear_plan(int pieces, bool mx8, int m, int n, int k)
{
    if (k == 0 || (!mx8 && k < 8)) return {Mx4LinearPlan::FewTerms, 0, 0, 0, 0, 0};
    // Up to two tiles a workgroup; more rows of X read B again (four would take too many registers: 64 x
    // 8192 x 8192 bf16 27.9 us against 24.9).
    Mx4LinearPlan p = {Mx4LinearPlan::Rows, 16, m <= 16 ? 1 : 2, 2, 4, 1};
    if (m <= 2) {
        p.tokens = 2;
        p.tiles = 1;
    } else if (pieces > 1 && m <= 8) {
        p.tokens = 8;
        p.tiles = 1;
    } else if (pieces > 1) {
        // Past one round of those workgroups (two to a CU; one of fp16's two tiles) the other kernel, which takes four
        // times the rows of B a workgroup: fp16 16 x 17000 x 8192 32.6 us against 39.7, but 16 x 12000 x 8192 32.0 against 27.5;
        // fp32 17 x 8192 x 8192 38.5 against 34.9, but 20 x 9000 x 8192 39.1 against 52.8.
        const bool two = pieces == 2 && m > 16;
        const int64_t others = (int64_t)((n + 31) / 32) * ((m + (two ? 31 : 15)) / (two ? 32 : 16));
        if (n > 16 * 256 && others > (two ? 256 : 512)) return {Mx4LinearPlan::Tall, 0, 0, 0, 0, 0};
        if (pieces == 3) {  // (three pieces of 16 tokens would not fit the LDS)
            p.tokens = 8;
            p.tiles = 2;
        }
    }
    if (n <= 16 * 256) {
        // one block of B's rows a workgroup, of which a CU has one: eight waves (1 x 4096 x 16384 9.8 us, by
        // four 12.2)
        p.blocks = 1;
        p.waves = 8;
    } else if (m <= 2 && pieces == 1) {
        // several workgroups to a CU, of four waves: one's loads go on while another adds up (1 x 28672
        // x 8192, groups in order, 26.5 us, by eight 28.9).  Two blocks each (16 x 28672 x 8192 38 us, one 45), but for one
        // token of one piece (28.7 against 26.5; 12000 x 4096 8.7 against 7.6)
        p.blocks = 1;
    }
    // One group of terms under way (1 x 12000 x 4096 bf16 7.3 us, with two 7.9; 16 x 12000 x 4096 of 8 bits 11.2 and
    // 12.1; fp32 1 x 20000 x 6000 17.3 and 20.4, 8 x 8192 x 4096 10.3 and 11.1); of one token in one piece
    // two where a wave has eight turns (2 x 8192 x 16384 16.1, with one 17.7; 1 x 28672 x 8192 24.1 and 24.7; but
    // 1 x 16384 x 8192 15.3 and 14.7).  Three and four are slower.
    if (m <= 2 && pieces == 1 && k > 7 * 256 * p.waves) p.ahead = 2;
    return p;
}

// A mixture is computed for 64 tokens at a time (kernels' z): tokens of other chunks share no tile.
constexpr int kMoeChunk = 64;
constexpr int kTileWaves = 4;
// Up to so many tokens and experts the first product's workgroups choose, too: 1 us where a launch costs 4.
constexpr int kFewTokens = 8, kFewExperts = 64;

struct Mx4MoePlan {
    bool one;   // a token: up_one_kernel and down_one_kernel
    bool few;   // the first product's workgroups choose
    int each;   // of the choice, logits to a lane
    int up, down;            // tokens to a tile of the first product and of the second
    bool up_rows, down_rows;  // rows for each wave (TileProduct without SPLIT)
    unsigned chunks, up_tiles, down_tiles;  // of a chunk: at most
};

inline Mx4MoePlan mx4_moe_plan(int pieces, int tokens, int width, int hidden, int experts, int topk)
{
    Mx4MoePlan p = {};
    p.one = tokens == 1;
    p.each = experts <= 64 ? 1 : experts <= 128 ? 2 : 8;
    if (p.one) return p;
    const int chunk = tokens < kMoeChunk ? tokens : kMoeChunk, choices = chunk * topk;
    p.few = tokens <= kFewTokens && experts <= kFewExperts;
    // tiles of 16 where experts have more than 6 tokens on average, as most would need two of 8 (64 x 4096
    // x 2048, 4 of 32, fp16 113 against 120 us, fp32 124 against 130; 24 tokens of it 106 against 98 and 118
    // against 99)
    const bool many = !p.few && choices > 6 * experts;
    p.up = many || pieces == 1 ? 16 : 8;
    p.down = many ? 16 : 8;
    auto most = [&](int size) {
        return (unsigned)(experts + choices / size < choices ? experts + choices / size : choices);
    };
    p.chunks = (unsigned)((tokens + kMoeChunk - 1) / kMoeChunk);
    p.up_tiles = most(p.up);
    p.down_tiles = most(p.down);
    // Rows for each wave from so many workgroups on.  Of 1, 100, 200, 300 and never, at 11 sizes of each type, 200
    // is the best or within 5 % of it at 28 of 33 and 14 % off at most; from 1 on, 200 and never, us in a graph:
    //   bf16 2 x 2048 x 1024, 2 of 8 25.4, 19.4, 19.4;  3 of it, 3 of 16 26.0, 23.0, 23.5;  4 x 1024 x 2048, 2 of 8
    //   26.1, 21.4, 23.8;  12 x 1024 x 1024, 2 of 16 24.3, 23.7, 26.5;  2 x 4096 x 2048, 4 of 32 37.4, 38.1, 44.7;
    //   fp16 4 x 4096 x 2048, 2 of 8 39.1, 40.2, 35.4;  fp32 8 x 1500 x 700, 2 of 16 26.8, 28.3, 28.8
    constexpr int64_t ENOUGH = 200;
    const int64_t up_wide = (hidden + 255) / 256 * 4, down_wide = ((width + 31) / 32 + kTileWaves - 1) / kTileWaves;
    p.up_rows = up_wide * p.up_tiles * p.chunks >= ENOUGH;
    p.down_rows = down_wide * p.down_tiles * p.chunks >= ENOUGH;
    return p;
}

}  // namespace sbx
