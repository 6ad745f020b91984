"""GPU tests of sbx_mx4_gemm against the plain implementation in 64 bits.

Elements are multiples of 1/2 up to 6 and codes lie within 2 of each other, so
terms are multiples of a 2^-2 quantum up to 36 * 2^4 of it: sums of fewer than
2^24 / (144 * 16) = 7281 of them are exact in 32 bits whatever their order,
and results have to be equal after the one rounding to their type.  Where codes
are spread over more, sums round: the error is held to 1e-5 of the result in
the 2-norm, as for the library's fp32 products.
"""
import numpy as np
import pytest

import mx4_reference as ref

pytestmark = pytest.mark.gpu

TYPES = ["f32", "bf16", "f16"]


def _types(name):
    import torch
    import sushiblas_amd as sbx
    return {"f32": (torch.float32, sbx.F32), "bf16": (torch.bfloat16, sbx.BF16),
            "f16": (torch.float16, sbx.F16)}[name]


def _codes(rng, rows, k, lo=126, hi=129):
    nb = (k + 31) // 32
    n = rng.integers(0, 16, (rows, nb, 32)).astype(np.uint8)
    # past the last term: zeros, as the quantiser leaves them
    n.reshape(rows, nb * 32)[:, k:] = 0
    return n, rng.integers(lo, hi, (rows, nb)).astype(np.uint8)


def _operand(cuda, n, sc, pp=0, ps=0, fill=0xFF):
    """Packed on the device; what lies beside the matrix, codes past the last
    block among it, is 0xFF (NaN, were it used)."""
    import torch
    rows, nb = sc.shape
    P, S = ref.pack(n, sc, ldp=16 * (nb + pp), lds=8 * (rows + ps), fill=fill)
    if nb % 8:
        S[-1, :8 * rows].reshape(rows, 8)[:, nb % 8:] = fill
    return torch.from_numpy(P).to(cuda), torch.from_numpy(S).to(cuda)


def _run(cuda, name, m, n, k, alpha=1.0, beta=0.0, relu=False, layout=0, pads=(0, 0, 0, 0, 0), lo=126, hi=129,
         stream=None, exact=True, seed=0):
    import torch
    import sushiblas_amd as sbx
    dt, code = _types(name)
    rng = np.random.default_rng(m * 131 + n * 17 + k + seed)
    a, b = _codes(rng, m, k, lo, hi), _codes(rng, n, k, lo, hi)
    A, SA = _operand(cuda, *a, pads[0], pads[1])
    B, SB = _operand(cuda, *b, pads[2], pads[3])
    # C: small integers, or NaN where it must not be read
    rows, cols = (m, n) if layout == 0 else (n, m)
    C = torch.from_numpy(rng.integers(-8, 9, (rows, cols + pads[4])).astype(np.float32)).to(dt)
    C0 = C.clone()
    if beta == 0:
        C[:, :cols] = float("nan")
    dC = C.to(cuda)
    torch.cuda.synchronize()
    print("mx4_gemm", name, m, n, k, alpha, beta, relu, layout, pads, flush=True)
    sbx.mx4_gemm(code, layout, m, n, k, alpha, A, A.shape[1], SA, SA.shape[1], B, B.shape[1], SB, SB.shape[1],
                 beta, dC, cols + pads[4], epilogue=sbx.EPILOGUE_RELU if relu else sbx.EPILOGUE_NONE,
                 stream=stream)
    torch.cuda.synchronize()
    want = alpha * (ref.values(*a, k) @ ref.values(*b, k).T)
    if layout == 1:
        want = want.T
    want = want + beta * C0[:, :cols].double().numpy()
    if relu:
        want = np.maximum(want, 0.0)
    got = dC.cpu()
    assert torch.equal(got[:, cols:], C0[:, cols:])
    if exact:
        w = torch.from_numpy(np.ascontiguousarray(want)).float().to(dt)  # want is exact in 32 bits
        assert torch.equal(got[:, :cols], w)
    else:
        g = got[:, :cols].double().numpy()
        assert np.linalg.norm(g - want) <= 1e-5 * np.linalg.norm(want)


# one row to several tiles of every size, ragged on all sides
SIZES = [(1, 1, 1), (1, 1, 32), (1, 17, 33), (2, 5, 128), (3, 300, 257), (16, 16, 256), (17, 65, 100),
         (32, 32, 512), (33, 31, 1000), (64, 64, 64), (65, 130, 300), (100, 1000, 96), (128, 128, 1024),
         (129, 257, 511), (255, 256, 768), (256, 256, 2048), (257, 513, 800), (512, 300, 1500), (8, 2000, 4096),
         (16, 1030, 2049), (37, 600, 5000), (700, 9, 320), (1, 5000, 7000), (640, 640, 640)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gemm_sizes(cuda, name, m, n, k):
    _run(cuda, name, m, n, k)


@pytest.mark.parametrize("m,n,k", [(1000, 1300, 520), (2048, 2048, 512), (2050, 2300, 130), (4097, 1025, 257),
                                   (512, 512, 7000), (300, 5000, 900), (64, 8192, 1024), (2304, 2304, 2304)])
def test_gemm_larger(cuda, m, n, k):
    _run(cuda, "f32", m, n, k)
    _run(cuda, "bf16", m, n, k, relu=True)


@pytest.mark.parametrize("m,n,k", [(600, 600, 31), (640, 577, 1000), (1025, 1000, 1700), (1500, 1500, 300),
                                   (450, 500, 6500), (1000, 1000, 4128), (1100, 1150, 2900), (129, 4096, 900),
                                   (1800, 2040, 1300), (3000, 3100, 200), (65, 65, 65), (4100, 4090, 96),
                                   (4090, 3001, 1090), (3001, 4090, 1090), (2049, 6000, 1030), (6000, 2100, 770)])
def test_gemm_tiles(cuda, m, n, k):
    """Few and many tiles of every kind, with terms that end inside a stage."""
    _run(cuda, "f16", m, n, k, beta=1.0)
    _run(cuda, "f32", m, n, k, layout=1)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("alpha,beta,relu", [(1.5, 0.0, False), (1.0, 1.0, False), (-0.5, 0.5, True),
                                             (0.0, 1.0, True), (0.0, 0.0, False)])
def test_gemm_scalars_and_layouts(cuda, name, layout, alpha, beta, relu):
    for m, n, k in ((5, 70, 300), (130, 200, 600), (300, 520, 260)):
        _run(cuda, name, m, n, k, alpha, beta, relu, layout)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("pads", [(1, 0, 0, 0, 1), (0, 1, 3, 0, 8), (2, 5, 1, 3, 3)])
def test_gemm_leading_dimensions(cuda, name, pads):
    for m, n, k in ((3, 90, 290), (70, 81, 1000), (300, 270, 513)):
        _run(cuda, name, m, n, k, beta=1.0, pads=pads)


@pytest.mark.parametrize("m,n,k", [(4, 300, 3000), (130, 140, 2000), (520, 600, 1024), (2048, 2048, 1000)])
def test_gemm_wide_scales(cuda, m, n, k):
    """Codes over 2^12 of range: sums round."""
    _run(cuda, "f32", m, n, k, lo=110, hi=122, exact=False)


def test_gemm_small_results(cuda):
    """Scales whose products lie near fp32's smallest normal numbers, still exact."""
    _run(cuda, "f32", 40, 50, 300, lo=66, hi=68)
    _run(cuda, "f32", 300, 300, 300, lo=66, hi=68)


def test_gemm_no_terms(cuda):
    """k = 0 and alpha = 0: C = beta * C, operands not looked at."""
    import torch
    import sushiblas_amd as sbx
    for name in TYPES:
        dt, code = _types(name)
        c0 = torch.arange(-30, 30, dtype=torch.float32).reshape(6, 10).to(dt)
        for k, alpha in ((0, 1.0), (64, 0.0)):
            c = c0.to(cuda)
            sbx.mx4_gemm(code, 0, 6, 10, k, alpha, None, 0, None, 0, None, 0, None, 0, 0.5, c, 10,
                         epilogue=sbx.EPILOGUE_RELU)
            assert torch.equal(c.cpu(), (c0.float() * 0.5).clamp_min(0).to(dt))


@pytest.mark.parametrize("m,n,k", [(3, 200, 700), (130, 100, 300), (300, 400, 520)])
def test_gemm_nan_blocks(cuda, m, n, k):
    """A NaN block makes its row (A) or column (B) NaN, and nothing else."""
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(4)
    a, b = _codes(rng, m, k), _codes(rng, n, k)
    a[1][m - 1, 3], b[1][7, -1], b[1][n - 1, 0] = 255, 255, 255
    A, SA = _operand(cuda, *a)
    B, SB = _operand(cuda, *b)
    C = torch.zeros((m, n), device=cuda)
    sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, A, A.shape[1], SA, SA.shape[1], B, B.shape[1], SB, SB.shape[1], 0.0, C, n)
    want = ref.values(*a, k) @ ref.values(*b, k).T
    nan = np.zeros((m, n), dtype=bool)
    nan[m - 1], nan[:, 7], nan[:, n - 1] = True, True, True
    got = C.cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), nan)
    np.testing.assert_array_equal(got[~nan], want[~nan].astype(np.float32))


def test_gemm_operand_parts(cuda):
    """Rows and 256-element column groups of larger matrices, by pointer and leading dimension."""
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(6)
    a, b = _codes(rng, 200, 1024), _codes(rng, 333, 1024)
    A, SA = _operand(cuda, *a)
    B, SB = _operand(cuda, *b)
    for r0, m, g, k in ((5, 100, 1, 512), (1, 7, 2, 300), (77, 123, 3, 256)):
        C = torch.empty((m, 333), device=cuda)
        sbx.mx4_gemm(sbx.F32, 0, m, 333, k, 1.0, A[r0:, 128 * g:], A.shape[1], SA[g:, 8 * r0:], SA.shape[1],
                     B[:, 128 * g:], B.shape[1], SB[g:], SB.shape[1], 0.0, C, 333)
        va = ref.values(*a, 1024)[r0:r0 + m, 256 * g:256 * g + 256 * 4]
        vb = ref.values(*b, 1024)[:, 256 * g:]
        # terms past k within the last block count: the operand is cut at a block
        kk = min((k + 31) // 32 * 32, va.shape[1])
        np.testing.assert_array_equal(C.cpu().numpy(), (va[:, :kk] @ vb[:, :kk].T).astype(np.float32))


def test_gemm_is_deterministic(cuda):
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(8)
    for m, n, k in ((8, 512, 8192), (256, 256, 16384), (1000, 1000, 3000)):
        a, b = _codes(rng, m, k, 100, 130), _codes(rng, n, k, 100, 130)
        A, SA = _operand(cuda, *a)
        B, SB = _operand(cuda, *b)
        outs = []
        for _ in range(3):
            C = torch.empty((m, n), device=cuda)
            sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, A, A.shape[1], SA, SA.shape[1], B, B.shape[1], SB, SB.shape[1],
                         0.0, C, n)
            outs.append(C)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_gemm_past_32_bit_offsets(cuda):
    """Operand rows, code groups and C rows whose byte offsets pass 32 bits."""
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(9)
    m, n, k = 600, 5, 600
    a, b = _codes(rng, m, k), _codes(rng, n, k)
    A, SA = _operand(cuda, *a)
    B, SB = _operand(cuda, *b)
    ld = (1 << 23) - 16
    far = torch.empty(m * ld, dtype=torch.uint8, device=cuda)
    torch.as_strided(far, A.shape, (ld, 1)).copy_(A)
    lds = (1 << 32) - 16
    fars = torch.empty(3 * lds, dtype=torch.uint8, device=cuda)
    torch.as_strided(fars, SA.shape, (lds, 1)).copy_(SA)
    want = (ref.values(*a, k) @ ref.values(*b, k).T).astype(np.float32)
    ldc = 2_000_000
    C = torch.empty(m * ldc, device=cuda)
    sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, far, ld, fars, lds, B, B.shape[1], SB, SB.shape[1], 0.0, C, ldc)
    np.testing.assert_array_equal(torch.as_strided(C, (m, n), (ldc, 1)).cpu().numpy(), want)
    C = torch.empty((n, m), device=cuda)
    sbx.mx4_gemm(sbx.F32, 0, n, m, k, 1.0, B, B.shape[1], SB, SB.shape[1], far, ld, fars, lds, 0.0, C, m)
    np.testing.assert_array_equal(C.cpu().numpy(), want.T)


@pytest.mark.parametrize("m,n,k", [(4, 1000, 4096), (300, 300, 4096), (700, 700, 512)])
def test_gemm_on_another_stream_and_in_a_graph(cuda, m, n, k):
    import torch
    import sushiblas_amd as sbx
    _run(cuda, "bf16", m, n, k, stream=torch.cuda.Stream())
    rng = np.random.default_rng(10)
    ops = [_operand(cuda, *_codes(rng, m, k)) for _ in range(4)]
    A, SA = (t.clone() for t in ops[0])
    B, SB = _operand(cuda, *_codes(rng, n, k))
    C, want = torch.empty((m, n), device=cuda), torch.empty((m, n), device=cuda)

    def call(C):
        sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, A, A.shape[1], SA, SA.shape[1], B, B.shape[1], SB, SB.shape[1],
                     0.0, C, n)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call(C)  # the stream has its workspace before the capture
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call(C)
    for P, S in ops[1:]:
        A.copy_(P)
        SA.copy_(S)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call(want)
        torch.cuda.synchronize()
        assert torch.equal(C, want)
