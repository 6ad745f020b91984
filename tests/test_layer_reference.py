"""CPU checks of the plain implementations that the norm's, the few-token layer's and the
mixture's GPU tests compare with."""
import numpy as np
import pytest
import torch

import layer_reference as ref


def test_e4m3_is_torchs():
    n = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(n).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ref.e4m3_values(), t)
    fine = ~np.isnan(t)
    np.testing.assert_array_equal(ref.e4m3_byte(t[fine]), n[fine])
    a = np.random.default_rng(1).normal(size=20000) * np.exp2(np.random.default_rng(2).integers(-11, 9, 20000))
    a = np.clip(a.astype(np.float32).astype(np.float64), -448, 448)
    near = torch.from_numpy(a).float().to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ref.e4m3(a), near)
    half = (t[fine][1:127] + t[fine][:126]) / 2  # ties
    near = torch.from_numpy(half).float().to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(ref.e4m3(half), near)


def test_quantize8_back():
    rng = np.random.default_rng(3)
    v = rng.normal(size=(5, 100)) * np.exp2(rng.integers(-30, 30, (5, 1)))
    v = v.astype(np.float32).astype(np.float64)
    n, code = ref.quantize8(v)
    back = ref.values8(n, code, 100)
    top = np.abs(np.pad(v, ((0, 0), (0, 28))).reshape(5, 4, 32)).max(-1).repeat(32, 1)[:, :100]
    # to the nearest, up to half a quantum of the largest, or by saturation 448 to 512
    assert (np.abs(back - v) <= np.maximum(np.abs(v) * 2.0 ** -4, top * 2.0 ** -17) + (np.abs(v) > 0.87 * top) * top / 8).all()


@pytest.mark.parametrize("eps", [1e-6, 0.5])
def test_gradient_against_differences(eps):
    rng = np.random.default_rng(4)
    h, w, dy = rng.normal(size=(3, 7)), rng.normal(size=7), rng.normal(size=(3, 7))
    dx, dw, _, _ = ref.norm_grad(h, w, eps, dy)
    loss = lambda h, w: (ref.norm(h, w, eps)[0] * dy).sum()  # noqa: E731
    d = 1e-5  # differences are off by d^2 and 2^-53 / d
    for i in np.ndindex(3, 7):
        e = np.zeros((3, 7))
        e[i] = d
        assert abs((loss(h + e, w) - loss(h - e, w)) / (2 * d) - dx[i]) < 1e-8
    for i in range(7):
        e = np.zeros(7)
        e[i] = d
        assert abs((loss(h, w + e) - loss(h, w - e)) / (2 * d) - dw[i]) < 1e-8


def test_route():
    x = np.array([[1.0, 0.0], [0.0, 1.0], [1.0, 1.0]])
    wr = np.array([[1.0, 0.0], [1.0, 2.0], [0.0, 2.0]])
    order, p, _ = ref.route(x, wr, 2, True)
    np.testing.assert_array_equal(order, [[0, 1], [1, 2], [1, 2]])
    np.testing.assert_allclose(p[0], [0.5, 0.5])
    _, q, _ = ref.route(x, wr, 2, False)
    np.testing.assert_allclose(q[0], np.exp([1, 1]) / np.exp([1, 1, 0]).sum())
    order, _, _ = ref.route(np.array([[np.nan, 0.0]]), wr, 3, True)
    np.testing.assert_array_equal(order, [[0, 1, 2]])


def test_moe_is_its_formula():
    rng = np.random.default_rng(5)
    x, wr = rng.normal(size=(2, 4)), rng.normal(size=(3, 4))
    w1, w2 = rng.normal(size=(3, 10, 4)), rng.normal(size=(3, 4, 5))
    y, off, order, p = ref.moe(x, wr, w1, w2, 1, True, 0.0)
    e = order[0, 0]
    z = torch.from_numpy(w1[e] @ x[0])
    want = w2[e] @ (torch.nn.functional.silu(z[:5]) * z[5:]).numpy()
    np.testing.assert_allclose(y[0], want, rtol=1e-12)
    assert (off > 0).all() and (p == 1).all()
