"""GPU tests of the few-token layer's forms, one by one, as layer_sizes.py lists them (and
test_layer_plan.py checks), against the plain implementation in 64 bits: results are equal
(test_mx4_linear_gpu.py)."""
import numpy as np
import pytest

import layer_reference as ref
import layer_sizes as sizes
from test_mx4_linear_gpu import _run

pytestmark = pytest.mark.gpu

NAMES = {p: n for n, p in sizes.PIECES.items()}


def _pad(k, apart):
    """Blocks beside B's rows that put them 4096 bytes apart, or a multiple, or not."""
    nb = -(-k // 32)
    return -nb % 256 if apart else int(nb % 256 == 0)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("m,n,k", [*sizes.TWO_AHEAD, *sizes.ONE_AHEAD])
def test_groups_under_way(cuda, apart, m, n, k):
    pads = (0, 0, 0, _pad(k, apart), 0)
    _run(cuda, "bf16", m, n, k, pads=pads)
    for name in ref.TYPES:
        _run(cuda, name, m, n, k, mx8=True, pads=pads)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("n,k", [(4100, 8192), (4200, 7700), (100, 16384)])
def test_rows_have_the_bits_that_they_have_alone(cuda, apart, mx8, n, k):
    """Two groups under way alone, one among three rows; and 20 rows in tiles of 16."""
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(k)
    wn, wc, _ = ref.random_mx4(rng, n, k, 110, 140)
    B, SB = ref.packed(cuda, wn, wc, _pad(k, apart))
    args = (B, B.shape[1], SB, SB.shape[1], 0.0)
    x, kw, alone = rng.normal(size=(20, k)) * np.exp2(rng.integers(-6, 7, (20, k))), {}, {}
    if mx8:
        xn, xc = ref.quantize8(x)
        X, S = (torch.from_numpy(v).to(cuda) for v in (xn.reshape(20, -1), ref.codes(xc)))
        kw = dict(SX=S, ldsx=S.shape[1])
    else:
        X = ref.padded(cuda, x, torch.bfloat16, 0)
    one = torch.zeros((20, n), device=cuda, dtype=torch.float32 if mx8 else torch.bfloat16)
    code = sbx.F32 if mx8 else sbx.BF16
    for i in range(20):
        if mx8:
            alone = dict(SX=S[:, 8 * i:], ldsx=S.shape[1])
        sbx.mx4_linear(code, 1, n, k, 1.0, X[i], X.shape[1], *args, one[i], n, **alone)
    for m in (2, 3, 20):
        Y = torch.zeros_like(one[:m])
        sbx.mx4_linear(code, m, n, k, 1.0, X, X.shape[1], *args, Y, n, **kw)
        assert torch.equal(Y, one[:m])


@pytest.mark.parametrize("pieces,m,n,k", [*sizes.TILES, *sizes.TALL])
def test_tiles(cuda, pieces, m, n, k):
    _run(cuda, NAMES[pieces], m, n, k)
    _run(cuda, NAMES[pieces], m, n, k, pads=(1, 0, 0, _pad(k, True), 1))
