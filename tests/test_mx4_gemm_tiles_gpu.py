"""GPU tests of every kernel of sbx_mx4_gemm (mx4_sizes.SIZES names them) where it can go
wrong: padded rows and code groups, C's other order and scalars, NaN blocks, operands
inside larger ones, the longest rows, scales far apart.

Sums are exact in 32 bits (see test_mx4_gemm_gpu.py), so results have to be equal."""
import numpy as np
import pytest

import mx4_reference as ref
from mx4_sizes import SIZES
from test_mx4_gemm_gpu import _codes, _operand, _run

pytestmark = pytest.mark.gpu

KERNELS = list(SIZES)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_leading_dimensions_and_scalars(cuda, kernel, name):
    _run(cuda, name, *SIZES[kernel], alpha=-0.5, beta=0.5, relu=True, pads=(2, 5, 1, 3, 3))


@pytest.mark.parametrize("kernel", KERNELS)
def test_column_major(cuda, kernel):
    """C's transpose in memory is the row-major product of B and A: its sizes choose the kernel."""
    n, m, k = SIZES[kernel]
    _run(cuda, "f32", m, n, k, alpha=2.0, layout=1, pads=(0, 1, 3, 0, 8))
    _run(cuda, "bf16", m, n, k, beta=1.0, layout=1, pads=(1, 0, 0, 2, 1))


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_blocks(cuda, kernel):
    """A NaN block makes its row (A) or column (B) NaN, and nothing else."""
    import torch
    import sushiblas_amd as sbx
    m, n, k = SIZES[kernel]
    rng = np.random.default_rng(4)
    a, b = _codes(rng, m, k), _codes(rng, n, k)
    a[1][m - 1, 3], a[1][0, -1], b[1][7, -1], b[1][n - 1, 0] = 255, 255, 255, 255
    A, SA = _operand(cuda, *a)
    B, SB = _operand(cuda, *b)
    C = torch.zeros((m, n), device=cuda)
    print("mx4_gemm", kernel, m, n, k, flush=True)
    sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, A, A.shape[1], SA, SA.shape[1], B, B.shape[1], SB, SB.shape[1], 0.0, C, n)
    nan = np.zeros((m, n), dtype=bool)
    nan[m - 1], nan[0], nan[:, 7], nan[:, n - 1] = True, True, True, True
    want = np.nan_to_num(ref.values(*a, k)) @ np.nan_to_num(ref.values(*b, k)).T
    got = C.cpu().numpy()
    np.testing.assert_array_equal(np.isnan(got), nan)
    np.testing.assert_array_equal(got[~nan], want[~nan].astype(np.float32))


@pytest.mark.parametrize("kernel", KERNELS)
def test_operand_parts(cuda, kernel):
    """Rows and 256-element column groups of larger matrices, by pointer and leading dimension."""
    import torch
    import sushiblas_amd as sbx
    m, n, k = SIZES[kernel]
    rng = np.random.default_rng(6)
    r0, g = 5, 1
    a, b = _codes(rng, m + r0 + 2, k + 600), _codes(rng, n + 3, k + 300)
    A, SA = _operand(cuda, *a)
    B, SB = _operand(cuda, *b)
    C = torch.empty((m, n), device=cuda)
    print("mx4_gemm", kernel, m, n, k, flush=True)
    sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, A[r0:, 128 * g:], A.shape[1], SA[g:, 8 * r0:], SA.shape[1], B, B.shape[1],
                 SB, SB.shape[1], 0.0, C, n)
    kk = -(-k // 32) * 32  # (terms past k within the last block count: the operand is cut at a block)
    va, vb = ref.values(*a, a[1].shape[1] * 32), ref.values(*b, b[1].shape[1] * 32)
    want = va[r0:r0 + m, 256 * g:256 * g + kk] @ vb[:n, :kk].T
    np.testing.assert_array_equal(C.cpu().numpy(), want.astype(np.float32))


@pytest.mark.parametrize("kernel", KERNELS)
def test_longest_rows(cuda, kernel):
    """Rows 2^23 - 16 bytes apart, so that 256 of them pass 2^31, and codes past 2^32."""
    import torch
    import sushiblas_amd as sbx
    m, n, k = SIZES[kernel]
    rng = np.random.default_rng(9)
    ops, vals = [], []
    for rows in (m, n):
        n_, sc = _codes(rng, rows, k)
        P, S = _operand(cuda, n_, sc)
        ld, groups = (1 << 23) - 16, S.shape[0]
        lds = (1 << 32) // (groups - 1) // 8 * 8 + 8
        far = torch.empty((rows - 1) * ld + P.shape[1], dtype=torch.uint8, device=cuda)
        torch.as_strided(far, P.shape, (ld, 1)).copy_(P)
        fars = torch.empty((groups - 1) * lds + S.shape[1], dtype=torch.uint8, device=cuda)
        torch.as_strided(fars, S.shape, (lds, 1)).copy_(S)
        ops.append((far, ld, fars, lds))
        vals.append(ref.values(n_, sc, k))
    C = torch.empty((m, n), device=cuda)
    print("mx4_gemm", kernel, m, n, k, flush=True)
    sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, *ops[0], *ops[1], 0.0, C, n)
    np.testing.assert_array_equal(C.cpu().numpy(), (vals[0] @ vals[1].T).astype(np.float32))
    del ops, far, fars
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kernel", KERNELS)
def test_scales_that_cancel(cuda, kernel):
    """Codes of every size whose two scales multiply to 2^-2 to 2^2; zero elements under the largest."""
    import torch
    import sushiblas_amd as sbx
    m, n, k = SIZES[kernel]
    rng = np.random.default_rng(12)
    a, b = _codes(rng, m, k), _codes(rng, n, k)
    nb = a[1].shape[1]
    c = rng.integers(4, 251, nb)
    a[1][:] = (c + rng.integers(-1, 2, (m, nb))).astype(np.uint8)
    b[1][:] = (254 - c + rng.integers(-1, 2, (n, nb))).astype(np.uint8)
    a[0][2], a[1][2], b[0][5], b[1][5] = 0, 254, 8, 254  # a row of 0, a row of -0
    a[0][:, 1], a[1][:, 1], b[0][:, 0], b[1][:, 0] = 0, 254, 0, 254
    A, SA = _operand(cuda, *a)
    B, SB = _operand(cuda, *b)
    C = torch.empty((m, n), device=cuda)
    sbx.mx4_gemm(sbx.F32, 0, m, n, k, 1.0, A, A.shape[1], SA, SA.shape[1], B, B.shape[1], SB, SB.shape[1], 0.0, C, n)
    want = ref.values(*a, k) @ ref.values(*b, k).T
    want[2], want[:, 5] = 0, 0
    np.testing.assert_array_equal(C.cpu().numpy(), want.astype(np.float32))
