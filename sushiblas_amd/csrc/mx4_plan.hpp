// mx4_plan.hpp -- which kernel an MXFP4 product runs (mx4_gemm.hip): plain arithmetic
// on its sizes (of the row-major C; a column-major one is its transpose), so that a
// host program can ask too.
#pragma once

#include <stdint.h>

namespace sbx {

enum class Mx4Kernel {
    Narrow2,  // up to 16 rows or columns, two blocks of 16 of the others a workgroup
    Narrow,   // the same, one block
    Tile64,
    Tile64Groups,   // two groups of waves that share the terms
    Tile128Stages,  // four stages
    Tile128,        // two workgroups to a CU
    Tile256x192,
    Tile192x256,
    Tile256,
    None  // no grid that a launch takes
};

// The kernels' times, in us, for choosing one: a launch and, for each round of `per_cu` workgroups
// on each CU, `fixed` (the first stage's arrival, and the results' way out) and `step` per `terms`
// terms, fitted to the times beside (bf16 results; * fp32).  The 256^2 tile asks the L2s for half
// of what 128^2 does, and 128^2 for half of 64^2; what counts for few tiles is a stage's latency,
// that more stages, groups of waves or workgroups on a CU hide: four of the 64^2 with one group
// fit on one.  Three quarters of a 256^2 tile use all CUs where whole ones leave a quarter idle.
//                   512^3  1024^2  1024^2  2048^2  4096 x 1024  4096^2  4096^3  4095 x 3001  6000^2
//                          x 2048  x 8192   x 512       x 4096  x 1024               x 2047  x 1000
//   64^2, 1 group     4.5     7.1    16.2     8.1         18.4
//   64^2, 2 groups    5.1     7.1    13.5    16.7         29.3    62.4   105.2
//   128^2, 4 stages   6.0     8.4    21.0     7.5         15.2    25.3    50.7
//   128^2, 2 per CU   7.1    10.2    26.3     8.3         17.2    20.6    43.7        31.6*    43.8
//   256 x 192                                                                         27.9*    45.7
//   192 x 256                                                                                  40.6
//   256^2                            45.4                 28.3    16.7    36.2        31.9*    46.4
struct Mx4TilePlan {
    Mx4Kernel kernel;
    int rows, cols, per_cu, terms;
    double step, fixed;
};
constexpr Mx4TilePlan kMx4TilePlans[] = {
    {Mx4Kernel::Tile64, 64, 64, 1, 256, 0.39, 1.2},
    {Mx4Kernel::Tile64, 64, 64, 2, 256, 0.55, 2.0},
    {Mx4Kernel::Tile64, 64, 64, 4, 256, 0.75, 3.3},
    {Mx4Kernel::Tile64Groups, 64, 64, 1, 512, 0.53, 2.3},
    {Mx4Kernel::Tile128Stages, 128, 128, 1, 256, 0.56, 3.3},
    {Mx4Kernel::Tile128, 128, 128, 2, 256, 0.95, 4.7},
    {Mx4Kernel::Tile256x192, 256, 192, 1, 256, 1.18, 10.5},
    {Mx4Kernel::Tile192x256, 192, 256, 1, 256, 1.12, 9.5},
    {Mx4Kernel::Tile256, 256, 256, 1, 256, 1.45, 10.0}};
constexpr double kMx4LaunchUs = 2.5;
constexpr int kMx4Cus = 256;
constexpr double kMx4Never = 1e30;

inline double mx4_tile_us(const Mx4TilePlan& t, int m, int n, int k)
{
    auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    const int64_t tiles = up(m, t.rows) * up(n, t.cols), rounds = up(tiles, t.per_cu * kMx4Cus);
    if (tiles * 512 > 0xffffffff) return kMx4Never;  // threads: more than a launch takes
    return kMx4LaunchUs + (double)rounds * (t.fixed + (double)up(k, t.terms) * t.step);
}

inline Mx4Kernel mx4_kernel(int m, int n, int k)
{
    const int narrow = m < n ? m : n, wide = m < n ? n : m;
    // One narrow block: the wide operand at the rate memory gives it.  Two blocks of it a
    // workgroup where that leaves one for each CU (1 x 8192 x 8192: 9.2 against 9.5 us, 16 rows
    // 10.3 against 11.7; the 64^2 tile 11.5 and 11.2).
    if (narrow <= 16) return wide > 16 * kMx4Cus ? Mx4Kernel::Narrow2 : Mx4Kernel::Narrow;
    double best = kMx4Never;
    Mx4Kernel pick = Mx4Kernel::None;
    for (const Mx4TilePlan& t : kMx4TilePlans) {
        const double us = mx4_tile_us(t, m, n, k);
        if (us < best) {
            best = us;
            pick = t.kernel;
        }
    }
    if (pick == Mx4Kernel::None) return pick;
    // Small results over many terms (256^2 x 8192: 6.6 against 10.9 us on the 64^2 tile, 128 x 1024 x
    // 8192 10.8 against 10.8): up to 2048 terms of a block, none among them, take its waves about 1 us.
    const double blocks = ((narrow + 15) / 16) * (double)((wide + 15) / 16) / kMx4Cus;
    const int steps = k > 0 ? (k + 2047) / 2048 : 1;
    return 2.2 + steps * (blocks < 1 ? 1 : blocks) < best ? Mx4Kernel::Narrow : pick;
}

}  // namespace sbx
