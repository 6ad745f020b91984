"""GPU tests of the MXFP4 operators on tensors whose dimensions of one entry have
torch's own strides: one group of codes (up to 256 terms) as contiguous() leaves
it.  Values against the plain implementation, equal (see test_mx4_gemm_gpu.py)."""
import numpy as np
import pytest

import mx4_reference as ref

pytestmark = pytest.mark.gpu


def _codes_room(cuda, rows, cols):
    import torch
    groups = -(-cols // 256)
    return torch.full((rows, groups, 8), 0xA5, dtype=torch.uint8, device=cuda).permute(1, 0, 2).contiguous()


def _operand(cuda, rng, rows, k):
    """Values (rows x k, float64) and their packed form, codes by way of contiguous()."""
    import torch
    nb = -(-k // 32)
    n = rng.integers(0, 16, (rows, nb, 32)).astype(np.uint8)
    n.reshape(rows, nb * 32)[:, k:] = 0
    sc = rng.integers(126, 129, (rows, nb)).astype(np.uint8)
    P, S = ref.pack(n, sc)
    room = _codes_room(cuda, rows, k)
    room.copy_(torch.from_numpy(S).reshape(room.shape))
    return ref.values(n, sc, k), torch.from_numpy(P).to(cuda), room


TERMS = [1, 31, 32, 255, 256]


def _product(cuda, m, n, k):
    import torch
    import sushiblas_amd as sbx
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, A, SA = _operand(cuda, rng, m, k)
    b, B, SB = _operand(cuda, rng, n, k)
    c0 = rng.integers(-8, 9, (m, n))
    C = torch.from_numpy(c0).float().to(cuda)
    print("mx4_gemm", m, n, k, SA.stride(), flush=True)
    sbx.mx4_gemm(sbx.F32, 0, m, n, k, 0.5, A, A.stride(0), SA, SA.stride(0), B, B.stride(0), SB, SB.stride(0),
                 1.0, C, C.stride(0))
    np.testing.assert_array_equal(C.cpu().numpy(), (0.5 * (a @ b.T) + c0).astype(np.float32))


@pytest.mark.parametrize("k", TERMS)
def test_product_of_one_group(cuda, k):
    _product(cuda, 500, 520, k)


@pytest.mark.parametrize("k", TERMS + [700])
@pytest.mark.parametrize("m,n", [(1, 5000), (3, 40), (4501, 1), (60, 70), (16, 4110)])
def test_product_of_one_group_or_row_narrow(cuda, m, n, k):
    """On the kernel for narrow operands, whose last workgroup has few of the wide one's rows."""
    _product(cuda, m, n, k)


@pytest.mark.parametrize("cols", TERMS)
def test_quantize_and_back_one_group(cuda, cols):
    import torch
    import sushiblas_amd as sbx
    rows = 70
    x = torch.randn((rows, cols), generator=torch.Generator().manual_seed(cols))
    P = torch.empty((rows, 16 * -(-cols // 32)), dtype=torch.uint8, device=cuda)
    PT = torch.empty((cols, 16 * -(-rows // 32)), dtype=torch.uint8, device=cuda)
    S, ST = _codes_room(cuda, rows, cols), _codes_room(cuda, cols, rows)
    assert S.stride(0) == ST.stride(0) == 8
    print("quantize", rows, cols, flush=True)
    sbx.mx4_quantize(sbx.F32, rows, cols, x.to(cuda), cols, P, P.stride(0), S, S.stride(0), PT, PT.stride(0), ST,
                     ST.stride(0))
    for v, p, s in ((x.numpy(), P, S), (x.numpy().T, PT, ST)):
        wp, ws = ref.pack(*ref.quantize(v))
        np.testing.assert_array_equal(p.cpu().numpy(), wp)
        np.testing.assert_array_equal(s.cpu().numpy().reshape(ws.shape), ws)
        y = torch.empty(v.shape, device=cuda)
        sbx.mx4_dequantize(sbx.F32, *v.shape, p, p.stride(0), s, s.stride(0), y, y.stride(0))
        np.testing.assert_array_equal(y.cpu().numpy(), ref.fake(v))
