"""GPU tests of sbx_mx4_linear and sbx_mx4_moe at the ends of the scale codes: the largest MXFP4 values that
32 bits hold (codes 253 and 254), those past them, and MXFP8 values below bf16's least one."""
import numpy as np
import pytest

import layer_reference as ref
import mx4_reference as mx4
from test_mx4_moe_gpu import Mixture

pytestmark = pytest.mark.gpu

FORMS = [(1, 40, 40), (1, 300, 290), (2, 4200, 520), (1, 60, 9), (5, 40, 300), (16, 300, 600), (20, 33, 1000),
         (40, 4200, 290), (60, 4200, 1000), (9, 8300, 270)]


def _operands(cuda, name, mx8, m, k, rng):
    """X of 1 to 2 times 2^-20, as bf16 holds it, its values, and the arguments that say where it is."""
    import torch
    dt, _ = ref.types(name)
    nb = -(-k // 32)
    if not mx8:
        X = ref.padded(cuda, (1 + rng.integers(0, 8, (m, k)) / 8) * 2.0 ** -20, dt, 0)
        return X, ref.f64(X), {}
    n, code = rng.integers(56, 64, (m, nb, 32)).astype(np.uint8), np.full((m, nb), 107, np.uint8)  # from 1 on
    X, S = torch.from_numpy(n.reshape(m, 32 * nb)).to(cuda), torch.from_numpy(ref.codes(code)).to(cuda)
    return X, ref.values8(n, code, k), dict(SX=S, ldsx=S.shape[1])


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_largest_values(cuda, name, mx8, m, n, k):
    """Up to 1.5 2^127, in a block that the last term lies in: what follows it is not used, bit for bit."""
    import torch
    import sushiblas_amd as sbx
    dt, code = ref.types(name)
    rng = np.random.default_rng(m + n + k)
    wide, nb = 32 * (-(-k // 32)), -(-k // 32)
    wn, wc, _ = ref.random_mx4(rng, n, wide, 240, 246)
    wc[:, -1] = rng.integers(253, 255, n)
    flat = wn.reshape(n, wide)
    flat[:, 32 * (nb - 1):] = rng.integers(0, 4, (n, 32)) + 8 * rng.integers(0, 2, (n, 32))
    with_them, w = ref.packed(cuda, wn, wc), mx4.values(wn, wc, wide)[:, :k]
    flat[:, k:] = 0
    X, x, more = _operands(cuda, name, mx8, m, k, rng)
    got = []
    print("mx4_linear past the last term", name, mx8, m, n, k, flush=True)
    for B, SB in (with_them, ref.packed(cuda, wn, wc)):
        got.append(torch.zeros((m, n), dtype=dt, device=cuda))
        sbx.mx4_linear(code, m, n, k, 2.0 ** -110, X, X.shape[1], B, B.shape[1], SB, SB.shape[1], 0.0, got[-1], n, **more)
    torch.cuda.synchronize()
    assert torch.equal(*got)
    want, bound = 2.0 ** -110 * (x @ w.T), (k + 4) * 2.0 ** -134 * (np.abs(x) @ np.abs(w).T)
    assert (np.abs(ref.f64(got[0]) - want) <= bound + ref.HALF[name] * (np.abs(want) + bound) + ref.TINY[name]).all()


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (2, 4200, 320), (7, 300, 600), (40, 4200, 290)])
def test_values_past_32_bits_are_infinities(cuda, name, mx8, m, n, k):
    """In every third row of the weights: its results are not finite, others are as ever."""
    import torch
    import sushiblas_amd as sbx
    dt, code = ref.types(name)
    rng = np.random.default_rng(n + k)
    wn, wc, _ = ref.random_mx4(rng, n, k, 126, 129)
    wn[::3, 1, 3], wc[::3, 1] = 6, 253  # 2^128
    wn[::6, 1, 3], wc[::6, 1] = 4, 254
    w, (B, SB) = mx4.values(wn, wc, k), ref.packed(cuda, wn, wc)
    wide = torch.empty((n, k), device=cuda)
    sbx.mx4_dequantize(sbx.F32, n, k, B, B.shape[1], SB, SB.shape[1], wide, k)
    assert bool(torch.isinf(wide[::3, 35]).all())
    X, x, more = _operands(cuda, name, mx8, m, k, rng)
    Y = torch.zeros((m, n), dtype=dt, device=cuda)
    sbx.mx4_linear(code, m, n, k, 2.0 ** 20, X, X.shape[1], B, B.shape[1], SB, SB.shape[1], 0.0, Y, n, **more)
    torch.cuda.synchronize()
    got, others = ref.f64(Y), np.arange(n) % 3 > 0
    assert not np.isfinite(got[:, ~others]).any()
    want, bound = 2.0 ** 20 * (x @ w[others].T), (k + 4) * 2.0 ** -4 * (np.abs(x) @ np.abs(w[others]).T)
    assert (np.abs(got[:, others] - want) <= bound + ref.HALF[name] * (np.abs(want) + bound) + ref.TINY[name]).all()


@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,k", [(1, 50), (3, 300), (40, 40)])
def test_infinite_values_elsewhere(cuda, mx8, m, k):
    """Where x is 0, or behind the last term of their block: their rows' results are NaN; in blocks behind it
    they are not used."""
    import torch
    import sushiblas_amd as sbx
    rng, n, nb = np.random.default_rng(k), 60, -(-k // 32)
    wn, wc, _ = ref.random_mx4(rng, n, 32 * (nb + 1), 126, 129)
    wn[::3, nb - 1, 31], wc[::3, nb - 1] = 6, 253
    wn[1::3, 0, 3], wc[1::3, 0] = 7, 254
    wn[:, nb, :], wc[:, nb] = 7, 254
    w, (B, SB) = mx4.values(wn, wc, k), ref.packed(cuda, wn, wc)
    X, x, more = _operands(cuda, "f32", mx8, m, k, rng)
    X[:, 3], x[:, 3] = 0, 0
    Y = torch.zeros((m, n), device=cuda)
    sbx.mx4_linear(sbx.F32, m, n, k, 2.0 ** 20, X, X.shape[1], B, B.shape[1], SB, SB.shape[1], 0.0, Y, n, **more)
    torch.cuda.synchronize()
    got, others = ref.f64(Y), np.arange(n) % 3 == 2
    assert np.isnan(got[:, ~others]).all()
    want, bound = 2.0 ** 20 * (x @ w[others].T), (k + 4) * 2.0 ** -4 * (np.abs(x) @ np.abs(w[others]).T)
    assert (np.abs(got[:, others] - want) <= bound + ref.HALF["f32"] * (np.abs(want) + bound)).all()


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_mixture_with_values_past_32_bits(cuda, name, tokens):
    """In one expert's weights: tokens that chose it are not finite, the others' results keep their bits."""
    import torch
    width, hidden, experts, topk = 300, 200, 6, 2
    m = Mixture(cuda, name, width, hidden, experts)
    X = ref.padded(cuda, np.random.default_rng(tokens).normal(size=(tokens, width)), m.dt, 0)
    want, got = torch.zeros_like(X), torch.zeros_like(X)
    chosen = torch.zeros((tokens, topk), dtype=torch.int32, device=cuda)
    m.call(X, want, topk, True, chosen)
    e = int(chosen[0, 1])
    m.W2[e * width:(e + 1) * width, 0] = 0x66
    m.S2[0, 8 * e * width:8 * (e + 1) * width:8] = 253
    m.call(X, got, topk, True)
    torch.cuda.synchronize()
    has = (chosen == e).any(1)
    assert not bool(torch.isfinite(got[has]).any()) and torch.equal(got[~has], want[~has])
    assert bool(torch.isfinite(want).all())


@pytest.mark.parametrize("lo", [0, 1, 2, 3, 6])
@pytest.mark.parametrize("m", [1, 3, 20])
def test_smallest_values_of_8_bits(cuda, lo, m):
    """All elements under the least codes, each picked out by a weight of 2^100: what lies below 2^-133 is
    rounded, so a value is off by less than that (and from code 3 on, whose least bits are 2^-133, by nothing)."""
    import torch
    import sushiblas_amd as sbx
    xn = np.arange(256, dtype=np.uint8).reshape(1, 8, 32).repeat(m, 0)
    xn[(xn & 127) == 127] = 0
    xc = np.full((m, 8), lo, np.uint8)
    wn, wc = np.zeros((256, 8, 32), np.uint8), np.full((256, 8), 227, np.uint8)
    wn.reshape(256, 256)[np.arange(256), np.arange(256)] = 2
    B, SB = ref.packed(cuda, wn, wc)
    X, S = torch.from_numpy(xn.reshape(m, 256)).to(cuda), torch.from_numpy(ref.codes(xc)).to(cuda)
    Y = torch.zeros((m, 256), device=cuda)
    sbx.mx4_linear(sbx.F32, m, 256, 256, 1.0, X, 256, B, B.shape[1], SB, SB.shape[1], 0.0, Y, 256, SX=S, ldsx=S.shape[1])
    torch.cuda.synchronize()
    off = np.abs(ref.f64(Y) * 2.0 ** -100 - ref.values8(xn, xc, 256))
    assert (off < 2.0 ** -133).all() if lo < 3 else not off.any()
