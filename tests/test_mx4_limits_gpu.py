"""GPU tests of the MXFP4 operators on matrices so tall that their workgroups pass
2^32 threads: quantisation of 2^29 rows, products with 2^28 and 2^30.  Rows repeat a
short table's, so that results can be compared on the device, piece by piece."""
import numpy as np
import pytest

import mx4_reference as ref

pytestmark = pytest.mark.gpu

PERIOD = 4096


def _room(gib):
    import torch
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


def _repeats(t, table):
    """t's rows are table's (PERIOD of them), over and over."""
    import torch
    whole = t.shape[0] // PERIOD * PERIOD
    for at in range(0, whole, PERIOD << 12):
        part = t[at:min(at + (PERIOD << 12), whole)]
        if not bool((part.reshape(-1, *table.shape) == table).all()):
            return False
    return torch.equal(t[whole:], table[:t.shape[0] - whole])


def _table(cuda, seed):
    import torch
    return torch.randn((PERIOD, 1), generator=torch.Generator().manual_seed(seed)).bfloat16()


def test_quantize_tall(cuda):
    import torch
    import sushiblas_amd as sbx
    _room(30)
    rows = (1 << 29) + 5
    x = _table(cuda, 1)
    X = x.to(cuda).repeat(rows // PERIOD + 1, 1)[:rows].contiguous()
    P = torch.empty((rows, 16), dtype=torch.uint8, device=cuda)
    S = torch.empty((1, rows, 8), dtype=torch.uint8, device=cuda)
    nb = -(-rows // 32)
    PT = torch.empty((1, 16 * nb), dtype=torch.uint8, device=cuda)
    ST = torch.empty((-(-nb // 8), 1, 8), dtype=torch.uint8, device=cuda)
    print("quantize", rows, flush=True)
    sbx.mx4_quantize(sbx.BF16, rows, 1, X, 1, P, 16, S, 8 * rows, PT, 16 * nb, ST, 8)
    p, s = ref.pack(*ref.quantize(x.double().numpy()))
    assert _repeats(P, torch.from_numpy(p).to(cuda))
    assert _repeats(S[0], torch.from_numpy(s).reshape(PERIOD, 8).to(cuda))
    # along the column: whole tables, then 5 values of one (rows is 5 past a multiple of the period)
    p, s = ref.pack(*ref.quantize(x.double().numpy().T))
    whole = rows // PERIOD
    assert bool((PT[0, :whole * PERIOD // 2].reshape(whole, -1) == torch.from_numpy(p).to(cuda)).all())
    assert bool((ST[:whole * PERIOD // 256].reshape(whole, -1) == torch.from_numpy(s).reshape(1, -1).to(cuda)).all())
    p, s = ref.pack(*ref.quantize(x[:5].double().numpy().T))
    np.testing.assert_array_equal(PT[0, whole * PERIOD // 2:].cpu().numpy(), p[0])
    np.testing.assert_array_equal(ST[-1, 0].cpu().numpy(), s.reshape(-1))


@pytest.mark.parametrize("tall,narrow,layout,gib", [((1 << 28) + 40, 1, 1, 20), ((1 << 28) + 40, 3, 0, 20),
                                                    ((1 << 30) - 5, 20, 1, 90)])
def test_gemm_tall(cuda, tall, narrow, layout, gib):
    """C (tall x narrow in memory, by rows) of a tall operand and a narrow one."""
    import torch
    import sushiblas_amd as sbx
    _room(gib)
    rng = np.random.default_rng(narrow)

    def operand(rows):
        n = rng.integers(0, 16, (rows, 1, 32)).astype(np.uint8)
        sc = rng.integers(126, 129, (rows, 1)).astype(np.uint8)
        return ref.values(n, sc, 32), *(torch.from_numpy(t) for t in ref.pack(n, sc))

    a, A, SA = operand(PERIOD)
    b, B, SB = operand(narrow)
    times = tall // PERIOD + 1
    A, SA = A.to(cuda).repeat(times, 1)[:tall], SA.reshape(PERIOD, 8).to(cuda).repeat(times, 1)[:tall]
    B, SB = B.to(cuda), SB.to(cuda)
    C = torch.empty((tall, narrow), dtype=torch.bfloat16, device=cuda)
    print("mx4_gemm", tall, narrow, layout, flush=True)
    tall_op, narrow_op = (A, 16, SA, 8 * tall), (B, 16, SB, 8 * narrow)
    if layout == 0:
        sbx.mx4_gemm(sbx.BF16, 0, tall, narrow, 32, 1.0, *tall_op, *narrow_op, 0.0, C, narrow)
    else:  # the same memory as a narrow x tall matrix by columns
        sbx.mx4_gemm(sbx.BF16, 1, narrow, tall, 32, 1.0, *narrow_op, *tall_op, 0.0, C, narrow)
    assert _repeats(C, torch.from_numpy(a @ b.T).float().bfloat16().to(cuda))
