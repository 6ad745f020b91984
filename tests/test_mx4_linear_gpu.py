"""GPU tests of sbx_mx4_linear against the plain implementation in 64 bits.

Where x are small whole numbers and codes lie within 2 of each other, terms are multiples of one
quantum and fewer than 2^24 of it in sum, so results are equal after the one rounding to their
type whatever the order of the sums.  Elsewhere a sum of k terms in 32 bits is off by at most
(k + 4) 2^-24 of its terms' magnitudes, and rounded to its type once.  fp32 values lose what lies
below 2^-133, less than 2^-133 of each, which counts times the weight's magnitude."""
import numpy as np
import pytest

import layer_reference as ref
import mx4_reference as mx4

pytestmark = pytest.mark.gpu


def _run(cuda, name, m, n, k, alpha=1.0, beta=0.0, relu=False, mx8=False, pads=(0, 0, 0, 0, 0), exact=True, stream=None,
         x=None, codes=None, fill=float("nan")):
    """pads: of X (elements, or 16 bytes), SX, SB (rows), B (blocks), Y."""
    import torch
    import sushiblas_amd as sbx
    dt, code = ref.types(name)
    rng = np.random.default_rng(m * 131 + n * 17 + k)
    wn, wc, w = ref.random_mx4(rng, n, k, *((126, 129) if exact else (100, 150)))
    if codes is not None:
        wc = np.resize(codes, wc.shape).astype(np.uint8)
        w = mx4.values(wn, wc, k)
    B, SB = ref.packed(cuda, wn, wc, pads[3], pads[2])
    SX = None
    if mx8:
        v = rng.integers(-8, 9, (m, k)) if exact else rng.normal(size=(m, k)) * np.exp2(rng.integers(-6, 7, (m, k)))
        xn, xc = ref.quantize8(v if x is None else x)
        x = ref.values8(xn, xc, k)
        nb = xc.shape[1]
        X = np.full((m, 32 * nb + 16 * pads[0]), 0x7F, dtype=np.uint8)  # NaN
        X[:, :32 * nb] = xn.reshape(m, 32 * nb)
        S = ref.codes(xc, lds=8 * (m + pads[1]), fill=0xFF)
        if nb % 8:
            S[-1, :8 * m].reshape(m, 8)[:, nb % 8:] = 0xFF
        X, SX = torch.from_numpy(X).to(cuda), torch.from_numpy(S).to(cuda)
    else:
        if x is None:
            x = rng.integers(-8, 9, (m, k)) if exact else rng.normal(size=(m, k)) * np.exp2(rng.integers(-6, 7, (m, k)))
        X = ref.padded(cuda, x, dt, pads[0], fill)
        x = ref.f64(X)[:, :k]
    y0 = rng.integers(-8, 9, (m, n))
    Y = ref.padded(cuda, y0 if beta != 0 else np.full((m, n), np.nan), dt, pads[4], 7.0)
    torch.cuda.synchronize()
    print("mx4_linear", name, m, n, k, alpha, beta, relu, mx8, pads, flush=True)
    sbx.mx4_linear(code, m, n, k, alpha, X, X.shape[1], B, B.shape[1], SB, SB.shape[1], beta, Y, Y.shape[1], SX=SX,
                   ldsx=0 if SX is None else SX.shape[1], stream=stream,
                   epilogue=sbx.EPILOGUE_RELU if relu else sbx.EPILOGUE_NONE)
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore", over="ignore"):
        want = alpha * (x @ w.T) + (beta * y0 if beta != 0 else 0.0)
        bound = (k + 4) * 2.0 ** -24 * (abs(alpha) * (np.abs(x) @ np.abs(w).T) + np.abs(beta * y0))
        if name == "f32" and not mx8:
            bound = bound + abs(alpha) * 2.0 ** -133 * np.abs(w).sum(1)
    if relu:
        want = np.where(want > 0, want, 0.0)
    got = ref.f64(Y)
    assert (got[:, n:] == 7.0).all()
    got = got[:, :n]
    if exact:
        np.testing.assert_array_equal(got, ref.rounded_to(want, dt))
    else:
        # a result past the largest value of its type rounds to an infinity (next to it, either way)
        top = ref.TOP[name] * (1 + ref.HALF[name])
        want = np.where(np.abs(want) - bound > top, np.copysign(np.inf, want), want)
        fine = np.isfinite(want) & (np.isfinite(got) | (np.abs(want) + bound < top))
        np.testing.assert_array_equal(got[~np.isfinite(want)], want[~np.isfinite(want)])
        got, want, bound = got[fine], want[fine], bound[fine]
        assert (np.abs(got - want) <= bound + ref.HALF[name] * (np.abs(want) + bound) + ref.TINY[name]).all()
    return Y


# tokens from one to a few tiles of them, terms from one, ragged on all sides
SIZES = [(1, 1, 1), (1, 1, 32), (1, 17, 33), (2, 5, 128), (1, 300, 257), (3, 16, 256), (15, 65, 100), (16, 32, 512),
         (17, 31, 1000), (5, 64, 64), (31, 130, 300), (32, 1000, 96), (33, 257, 511), (48, 200, 768), (64, 256, 1024),
         (65, 70, 300), (8, 2000, 2040), (16, 1030, 2049), (1, 5000, 2300), (7, 640, 640), (1, 8193, 70), (4, 9000, 300),
         (100, 50, 260), (300, 40, 100), (1024, 20, 40), (18, 4100, 300), (33, 4225, 2049), (64, 4352, 1024), (200, 4130, 40)]


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes(cuda, name, m, n, k):
    _run(cuda, name, m, n, k)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes_of_8_bits(cuda, name, m, n, k):
    _run(cuda, name, m, n, k, mx8=True)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 300, 4096), (3, 4100, 1000), (16, 500, 8192), (33, 300, 2047), (64, 64, 5000)])
def test_far_magnitudes(cuda, name, mx8, m, n, k):
    _run(cuda, name, m, n, k, mx8=mx8, exact=False)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("alpha,beta,relu", [(1.5, 0.0, False), (1.0, 1.0, False), (-0.5, 0.5, True), (0.0, 1.0, True),
                                             (0.0, 0.0, False)])
def test_scalars(cuda, name, mx8, alpha, beta, relu):
    for m, n, k in ((1, 70, 300), (16, 33, 600), (40, 52, 260)):
        _run(cuda, name, m, n, k, alpha, beta, relu, mx8)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("pads", [(1, 1, 1, 1, 1), (8, 0, 0, 3, 8), (3, 2, 5, 0, 0)])
@pytest.mark.parametrize("m,n,k", [(1, 40, 100), (5, 300, 1000), (20, 33, 513)])
def test_strides(cuda, name, mx8, pads, m, n, k):
    _run(cuda, name, m, n, k, mx8=mx8, pads=pads)


def test_no_terms(cuda):
    import torch
    import sushiblas_amd as sbx
    for m, n in ((1, 70), (40, 300)):
        y = torch.full((m, n), 3.0, device=cuda)
        sbx.mx4_linear(sbx.F32, m, n, 0, 1.0, None, 0, None, 0, None, 0, 2.0, y, n)
        assert bool((y == 6.0).all())
        sbx.mx4_linear(sbx.F32, m, n, 0, 1.0, None, 0, None, 0, None, 0, 0.0, y, n)
        assert bool((y == 0.0).all())


@pytest.mark.parametrize("name", ref.TYPES)
def test_values_that_are_not_finite(cuda, name):
    """An infinity or NaN of x reaches the results that it is a term of (weights are not zero there);
    other rows keep theirs."""
    m, n, k = 6, 40, 600
    rng = np.random.default_rng(7)
    x = rng.integers(-8, 9, (m, k)).astype(np.float64)
    x[0, 5], x[2, 599], x[4, 300] = np.inf, np.nan, -np.inf
    import torch
    import sushiblas_amd as sbx
    dt, code = ref.types(name)
    wn, wc, w = ref.random_mx4(rng, n, k, 126, 129)
    wn = np.where(wn & 7 == 0, wn + 1, wn).astype(np.uint8)
    wn.reshape(n, -1)[:, k:] = 0
    w = mx4.values(wn, wc, k)
    wc = wc.copy()
    wc[3, 2] = 255  # a block that is NaN
    w[3, 64:96] = np.nan
    B, SB = ref.packed(cuda, wn, wc)
    X = ref.padded(cuda, x, dt, 0)
    Y = torch.zeros((m, n), dtype=dt, device=cuda)
    sbx.mx4_linear(code, m, n, k, 1.0, X, k, B, B.shape[1], SB, SB.shape[1], 0.0, Y, n)
    with np.errstate(invalid="ignore"):
        want = ref.rounded_to(x @ w.T, dt)
    np.testing.assert_array_equal(ref.f64(Y), want)


@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 7), (1, 9), (2, 31), (5, 33), (16, 250), (40, 262), (3, 319)])
def test_what_lies_past_the_last_term(cuda, mx8, m, k):
    """The first k columns of wider operands, X's others NaN: they count nowhere."""
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(100 * k + m)
    n, wide = 40, 320
    wn, wc, w = ref.random_mx4(rng, n, wide, 126, 129)
    B, SB = ref.packed(cuda, wn, wc)
    x, SX = rng.integers(-8, 9, (m, wide)), None
    if mx8:
        xn, xc = ref.quantize8(x)
        x = ref.values8(xn, xc, wide)
        X = xn.reshape(m, wide).copy()
        X[:, k:] = 0x7F
        X, SX = torch.from_numpy(X).to(cuda), torch.from_numpy(ref.codes(xc)).to(cuda)
    else:
        x = x.astype(np.float64)
        X = torch.from_numpy(x).float().to(cuda)
        X[:, k:] = float("nan")
    Y = torch.empty((m, n), device=cuda)
    sbx.mx4_linear(sbx.F32, m, n, k, 1.0, X, wide, B, B.shape[1], SB, SB.shape[1], 0.0, Y, n, SX=SX,
                   ldsx=0 if SX is None else SX.shape[1])
    np.testing.assert_array_equal(ref.f64(Y), x[:, :k] @ w[:, :k].T)


def test_smallest_and_largest_scales(cuda):
    """Codes at both ends; x of the other end, so that products are ordinary."""
    _run(cuda, "f32", 3, 40, 96, codes=[0, 1, 2], x=np.full((3, 96), 2.0 ** 120), exact=False)
    _run(cuda, "bf16", 3, 40, 96, codes=[0, 1, 2], x=np.full((3, 96), 2.0 ** 120), exact=False)
    _run(cuda, "f32", 3, 40, 96, codes=[250, 251, 252], x=np.full((3, 96), 1.7 * 2.0 ** -120), exact=False)
    _run(cuda, "bf16", 3, 40, 96, codes=[250, 251, 252], x=np.full((3, 96), 1.5 * 2.0 ** -120), exact=False)
    # values with bits far apart in 32
    x = np.float32(1 + 2.0 ** -23) * np.ones((3, 96), np.float32)
    _run(cuda, "f32", 3, 40, 96, x=x.astype(np.float64), exact=False)


def test_rows_have_the_bits_that_they_have_alone(cuda):
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(3)
    m, n, k = 37, 500, 3001
    wn, wc, _ = ref.random_mx4(rng, n, k, 110, 140)
    B, SB = ref.packed(cuda, wn, wc)
    for name in ref.TYPES:
        dt, code = ref.types(name)
        X = torch.from_numpy(rng.normal(size=(m, k))).to(dt).to(cuda)
        both = [torch.empty((m, n), dtype=dt, device=cuda) for _ in range(2)]
        args = (B, B.shape[1], SB, SB.shape[1], 0.0)
        sbx.mx4_linear(code, m, n, k, 1.0, X, k, *args, both[0], n)
        for i in range(m):
            sbx.mx4_linear(code, 1, n, k, 1.0, X[i], k, *args, both[1][i], n)
        assert torch.equal(both[0], both[1])


@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,n,k", [(60, 4200, 3001), (17, 4097, 260), (70, 4500, 8), (52, 4200, 1030)])
def test_rows_of_tall_weights(cuda, mx8, m, n, k):
    """Among many rows of X and of B: the same bits as alone."""
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(m)
    wn, wc, _ = ref.random_mx4(rng, n, k, 110, 140)
    B, SB = ref.packed(cuda, wn, wc)
    nb = -(-k // 32)
    for name in ref.TYPES:
        dt, code = ref.types(name)
        kw, alone = {}, {}
        if mx8:
            xn, xc = ref.quantize8(rng.normal(size=(m, k)) * np.exp2(rng.integers(-6, 7, (m, k))))
            X, S = (torch.from_numpy(v).to(cuda) for v in (xn.reshape(m, 32 * nb), ref.codes(xc)))
            kw = dict(SX=S, ldsx=S.shape[1])
        else:
            X = torch.from_numpy(rng.normal(size=(m, k)) * np.exp2(rng.integers(-6, 7, (m, k)))).to(dt).to(cuda)
        both = [torch.full((m, n + 3), 7.0, dtype=dt, device=cuda) for _ in range(2)]
        args = (B, B.shape[1], SB, SB.shape[1], 0.0)
        sbx.mx4_linear(code, m, n, k, 0.5, X, X.shape[1], *args, both[0], n + 3, **kw)
        for i in range(m):
            if mx8:  # (a row's codes are a run of 8 bytes in each group's)
                alone = dict(SX=S[:, 8 * i:], ldsx=S.shape[1])
            sbx.mx4_linear(code, 1, n, k, 0.5, X[i], X.shape[1], *args, both[1][i], n + 3, **alone)
        assert torch.equal(both[0], both[1])


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 300, 2049), (7, 40, 4000), (20, 100, 300), (64, 4352, 1100), (1, 4200, 3000),
                                   (3, 8200, 1500), (70, 4400, 2300), (12, 16500, 270), (2, 20, 8192)])
def test_rows_4096_bytes_apart(cuda, name, m, n, k):
    """Weights whose rows are so far apart, or a multiple: groups of terms in another order."""
    _run(cuda, name, m, n, k, pads=(0, 0, 0, 256 - -(-k // 32), 0))
    _run(cuda, name, m, n, k, mx8=True, pads=(0, 0, 0, 512 - -(-k // 32), 0))


@pytest.mark.parametrize("m,n,k", [(60, 4200, 3001), (17, 600, 2600), (70, 4500, 2050)])
def test_rows_4096_bytes_apart_have_the_bits_that_they_have_alone(cuda, m, n, k):
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(m)
    wn, wc, _ = ref.random_mx4(rng, n, k, 110, 140)
    B, SB = ref.packed(cuda, wn, wc, 256 - -(-k // 32))
    assert B.shape[1] == 4096
    for name in ref.TYPES:
        dt, code = ref.types(name)
        X = torch.from_numpy(rng.normal(size=(m, k)) * np.exp2(rng.integers(-6, 7, (m, k)))).to(dt).to(cuda)
        X[3, 5], X[m - 1, k - 1] = float("inf"), float("nan")
        both = [torch.empty((m, n), dtype=dt, device=cuda) for _ in range(2)]
        args = (B, B.shape[1], SB, SB.shape[1], 0.0)
        sbx.mx4_linear(code, m, n, k, 1.0, X, k, *args, both[0], n)
        for i in range(m):
            sbx.mx4_linear(code, 1, n, k, 1.0, X[i], k, *args, both[1][i], n)
        fine = ~torch.isnan(both[1])
        assert torch.equal(both[0][fine], both[1][fine]) and torch.equal(torch.isnan(both[0]), ~fine)
        assert bool(fine[:3].all()) and not bool(torch.isfinite(both[0][3]).any())


def test_another_stream_and_replays(cuda):
    import torch
    import sushiblas_amd as sbx
    _run(cuda, "bf16", 9, 1000, 700, stream=torch.cuda.Stream())
    rng = np.random.default_rng(5)
    wn, wc, _ = ref.random_mx4(rng, 300, 900)
    B, SB = ref.packed(cuda, wn, wc)
    x, y = torch.randn(5, 900, device=cuda), [torch.empty(5, 300, device=cuda) for _ in range(2)]

    def call(i):
        sbx.mx4_linear(sbx.F32, 5, 300, 900, 1.0, x, 900, B, B.shape[1], SB, SB.shape[1], 0.0, y[i], 300)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(1)
    for _ in range(3):
        x.copy_(torch.randn(5, 900, device=cuda))
        call(0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y[0], y[1])
