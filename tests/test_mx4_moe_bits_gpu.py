"""GPU tests of what sbx_mx4_moe holds between its two products: activations with the bits of 32.

Hidden units go in pairs whose results nearly cancel, so that a few bits of an activation are what
is left.  x are small whole numbers times powers of two, so the first product's sums are exact in 32
bits.  An activation takes expf (twice, 2^-23 each), and eight roundings of 2^-24 at most, its share's
among them: 2^-20 of it in all; pieces of 24 bits add 2^-22, and the second product's sums
(hidden + topk + 4) 2^-24 of their terms' magnitudes.  The result is rounded once."""
import numpy as np
import pytest

import layer_reference as ref
import mx4_reference as mx4
from test_mx4_moe_gpu import Mixture

pytestmark = pytest.mark.gpu


def paired(cuda, name, width, hidden, experts):
    """A mixture of hidden / 2 pairs an expert: the same gates, ups that differ in one element of the last
    column, opposite weights in the second product."""
    m = Mixture(cuda, name, width, hidden, experts)
    rng = np.random.default_rng(width + hidden)
    nb1, nb2 = -(-width // 32), -(-hidden // 32)
    n1 = rng.integers(0, 16, (experts, 2, hidden // 2, 2, nb1 * 32)).astype(np.uint8)
    n1[..., 1, :] = n1[..., 0, :]
    n1[:, 1, :, 0, width - 1], n1[:, 1, :, 1, width - 1] = 2, 3  # 1 and 1.5
    n1[..., width:] = 0
    n1 = n1.reshape(experts * 2 * hidden, nb1, 32)
    c1 = np.full((experts * 2 * hidden, nb1), 125 - int(np.log2(width) / 2), dtype=np.uint8)
    n2 = np.zeros((experts * width, nb2 * 32), dtype=np.uint8)
    half = rng.integers(1, 8, (experts * width, hidden // 2))
    n2[:, :hidden:2], n2[:, 1:hidden:2] = half, half + 8
    n2 = n2.reshape(experts * width, nb2, 32)
    c2 = np.full((experts * width, nb2), 126, dtype=np.uint8)
    m.w1 = mx4.values(n1, c1, width).reshape(experts, 2 * hidden, width)
    m.w2 = mx4.values(n2, c2, hidden).reshape(experts, width, hidden)
    m.W1, m.S1 = ref.packed(cuda, n1, c1)
    m.W2, m.S2 = ref.packed(cuda, n2, c2)
    return m


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("tokens,width,hidden,experts,topk", [(1, 600, 6, 8, 2), (1, 40, 12, 100, 3), (5, 600, 6, 8, 2),
                                                              (9, 300, 10, 70, 1), (40, 260, 8, 6, 2), (70, 64, 12, 8, 4)])
def test_activations_keep_32_bits(cuda, name, tokens, width, hidden, experts, topk):
    import torch
    m = paired(cuda, name, width, hidden, experts)
    rng = np.random.default_rng(tokens)
    x = rng.integers(-8, 9, (tokens, width)) * 0.25
    x[:, width - 1] = rng.integers(1, 9, tokens) * 2.0 ** -9
    X = ref.padded(cuda, x, m.dt, 0)
    x = ref.f64(X)
    Y = torch.zeros((tokens, width), dtype=m.dt, device=cuda)
    print("mx4_moe pairs", name, tokens, width, hidden, experts, topk, flush=True)
    m.call(X, Y, topk, True)
    torch.cuda.synchronize()
    order, p, _ = ref.route(x, m.wr, topk, True)
    y, off = np.zeros((tokens, width)), np.zeros((tokens, width))
    for t in range(tokens):
        for j in range(topk):
            z = m.w1[order[t, j]] @ x[t]
            a = z[:hidden] / (1 + np.exp(-z[:hidden])) * z[hidden:] * p[t, j]
            y[t] += m.w2[order[t, j]] @ a
            off[t] += np.abs(m.w2[order[t, j]]) @ np.abs(a) * (2.0 ** -20 + 2.0 ** -22 + (hidden + topk + 4) * 2.0 ** -24)
    got = ref.f64(Y)
    assert (np.abs(got - y) <= off + ref.HALF[name] * (np.abs(y) + off) + ref.TINY[name]).all()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 6, 70])
def test_silu_of_far_gates(cuda, name, tokens):
    """Gates from -160 to 90 with ups of 2^100: silu is of use as long as 32 bits hold its product with them,
    which is below exp(-88), where exp(-gate) passes their range."""
    import torch
    width, hidden = 16, 260
    m = Mixture(cuda, name, width, hidden, 2)
    n1, c1 = np.zeros((2, 2 * hidden, 1, 32), np.uint8), np.full((2, 2 * hidden, 1), 127, np.uint8)
    n1[:, np.arange(hidden), 0, np.arange(hidden) % 8] = 2  # the gates: x of one of the first 8 columns
    n1[:, hidden:, 0, 8] = 2
    c1[:, hidden:] = 227
    n2, c2 = np.zeros((2, width, 9, 32), np.uint8), np.full((2, width, 9), 127, np.uint8)
    n2[:, np.arange(width), 0, np.arange(width)] = 2  # a result: one unit of the hidden layer
    n1, c1, n2, c2 = n1.reshape(-1, 1, 32), c1.reshape(-1, 1), n2.reshape(-1, 9, 32), c2.reshape(-1, 9)
    m.w1 = mx4.values(n1, c1, width).reshape(2, 2 * hidden, width)
    m.w2 = mx4.values(n2, c2, hidden).reshape(2, width, hidden)
    m.W1, m.S1 = ref.packed(cuda, n1, c1)
    m.W2, m.S2 = ref.packed(cuda, n2, c2)
    x = np.zeros((tokens, width))
    x[:, :8] = -np.array([160, 130, 104, 100, 95, 90, 86, -90]) + np.arange(tokens)[:, None] % 4
    x[:, 8] = 1.0
    X = ref.padded(cuda, x, m.dt, 0)
    x = ref.f64(X)
    Y = torch.zeros((tokens, width), dtype=m.dt, device=cuda)
    m.call(X, Y, 1, True)
    torch.cuda.synchronize()
    order, _, _ = ref.route(x, m.wr, 1, True)
    want = np.empty((tokens, width))
    for t in range(tokens):
        z = m.w1[order[t, 0]] @ x[t]
        want[t] = m.w2[order[t, 0]] @ (z[:hidden] / (1 + np.exp(-z[:hidden])) * z[hidden:])
    # as above, one term a sum; pieces are of bf16, which ends at 2^-133
    off = np.abs(want) * (2.0 ** -20 + 2.0 ** -22 + 2.0 ** -23) + 2.0 ** -133
    got = ref.f64(Y)
    assert (np.abs(got - want) <= off + ref.HALF[name] * (np.abs(want) + off) + ref.TINY[name]).all()
