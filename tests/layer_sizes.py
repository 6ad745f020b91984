"""Sizes that reach each form of the few-token layer and of the mixture, for the tests that ask the
rule (csrc/layer_plan.hpp) and those that run them.  pieces: 1 of bf16 and MXFP8, 2 of fp16, 3 of fp32."""

PIECES = {"bf16": 1, "f16": 2, "f32": 3}

# m, n, k: with one piece, two groups of terms under way; (blocks of 16 rows, waves) to a workgroup
TWO_AHEAD = {(1, 4100, 8192): (1, 4), (2, 4200, 7700): (1, 4), (1, 100, 16384): (1, 8), (2, 40, 15001): (1, 8),
             (2, 4097, 7169): (1, 4), (1, 4096, 14337): (1, 8)}
# the same rows with one under way
ONE_AHEAD = {(1, 4100, 7168): (1, 4), (1, 4096, 14336): (1, 8), (3, 4100, 8192): (2, 4), (3, 100, 16384): (1, 8)}
# m, n, k by pieces: tokens to a tile and tiles to a workgroup
TILES = {(1, 16, 5000, 300): (16, 1), (1, 17, 5000, 300): (16, 2), (2, 2, 300, 300): (2, 1), (2, 8, 5000, 300): (8, 1),
         (2, 16, 5000, 300): (16, 1), (2, 17, 300, 300): (16, 2), (3, 8, 300, 300): (8, 1), (3, 9, 5000, 300): (8, 2),
         (3, 33, 4000, 300): (8, 2), (3, 2, 5000, 300): (2, 1)}
# pieces, m, n, k: the form for many rows of both
TALL = [(2, 16, 16600, 520), (2, 33, 4352, 1024), (2, 64, 4130, 2049), (3, 17, 8300, 520), (3, 40, 6000, 1300)]

# tokens, width, hidden, experts, topk: (rows for each wave in the first product, in the second), tokens to a
# tile of the second.  Several groups of 256 terms each, ragged and even ones.
ROWS = {(40, 1024, 512, 16, 4): (True, True, 16), (64, 1100, 1300, 16, 4): (True, True, 16),
        (7, 2049, 1030, 12, 4): (True, True, 8), (20, 1500, 700, 70, 4): (True, True, 8),
        (130, 600, 520, 6, 3): (True, True, 16), (9, 1100, 1300, 3, 1): (False, False, 8),
        (30, 600, 1300, 8, 2): (True, False, 16), (12, 2100, 300, 20, 2): (False, True, 8)}
# tokens, experts, topk: logits to a lane that chooses
CHOICES = {(1, 65, 8): 2, (1, 128, 8): 2, (1, 129, 16): 8, (1, 512, 16): 8, (1, 64, 8): 1, (9, 65, 4): 2, (9, 128, 8): 2,
           (9, 129, 8): 8, (3, 65, 4): 2, (3, 128, 3): 2, (12, 64, 6): 1}
