"""Sizes (m, n, k) that the MXFP4 product's rule (csrc/mx4_plan.hpp) gives to each of
its kernels, ragged on all sides, for the GPU tests; a CPU test holds the rule to it."""

SIZES = {
    "Narrow": (70, 81, 1000),
    "Narrow2": (3, 5000, 300),
    "Tile64": (500, 520, 300),
    "Tile64Groups": (300, 577, 4128),
    "Tile128Stages": (1000, 2100, 700),
    "Tile128": (2050, 2040, 300),
    "Tile256x192": (4090, 3001, 520),
    "Tile192x256": (2050, 4090, 520),
    "Tile256": (4100, 3001, 520),
}
