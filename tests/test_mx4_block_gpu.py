"""GPU tests of the feed-forward block of examples/mx4_feed_forward.py: dropout,
quantiser and product together, forward and backward.

Its values against the same formulas in 64 bits: a product's sums are exact in 32
bits here (see test_mx4_gemm_gpu.py), the inner matrices hold their type, so
results are the formulas' rounded once.
Its gradients against differences of the loss L = sum(G * Y): where X, W1, W2 and
G hold values that MXFP4 holds exactly along both axes, quantisation is the
identity, and L is linear in an entry of W2, and of W1 and X as long as no ReLU
switches; a difference of two values of L, whose terms are multiples of 2^-6 and
add up to less than 2^18, is then exact in 32 bits.
"""
import os
import sys

import numpy as np
import pytest

import mx4_reference as ref

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _block(tokens, width, hidden, p, dtype, seed=5):
    from mx4_feed_forward import FeedForward
    return FeedForward(tokens, width, hidden, p=p, seed=seed, dtype=dtype)


def _rounded(v, dtype):
    """v as the type holds it, in 64 bits."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(v)).float().to(dtype).double().numpy()


def _formulas(x, w1, w2, dy, p, seed, step, dtype):
    f = ref.fake
    h = _rounded(np.maximum(f(x) @ f(w1).T, 0.0), dtype)
    d = ref.dropped(h.astype(np.float32), p, seed, step).astype(np.float64)
    y = f(d) @ f(w2).T
    dd = _rounded(f(dy) @ f(w2.T).T, dtype)
    dz = ref.dropped(dd.astype(np.float32), p, seed, step, h.astype(np.float32)).astype(np.float64)
    return {"y": _rounded(y, dtype), "dx": _rounded(f(dz) @ f(w1.T).T, dtype),
            "dw1": _rounded(f(dz.T) @ f(x.T).T, np_f32()), "dw2": _rounded(f(dy.T) @ f(d.T).T, np_f32())}


def np_f32():
    import torch
    return torch.float32


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,width,hidden,p", [(1, 33, 70, 0.0), (7, 64, 96, 0.5), (48, 70, 130, 0.1),
                                                   (130, 257, 300, 0.2), (300, 512, 700, 0.1)])
def test_block_against_the_formulas(cuda, name, tokens, width, hidden, p):
    import torch
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]
    block = _block(tokens, width, hidden, p, dt)
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, width), generator=gen).to(dt)
    dy = (torch.randn((tokens, width), generator=gen) * 0.01).to(dt)
    print("block", name, tokens, width, hidden, p, flush=True)
    block.forward(x.to(cuda), step=3)
    block.backward(dy.to(cuda))
    want = _formulas(x.double().numpy(), block.w1.cpu().double().numpy(), block.w2.cpu().double().numpy(),
                     dy.double().numpy(), p, block.seed, 3, dt)
    for k, v in want.items():
        np.testing.assert_array_equal(getattr(block, k).cpu().double().numpy(), v, err_msg=k)


def _on_grid(rng, rows, cols):
    """Small values MXFP4 holds exactly along both axes: multiples of 1/2 up to 2 in magnitude
    beside a 2 in every block."""
    v = rng.integers(-4, 5, (rows, cols)) / 2.0
    v[::32, :] = 2.0
    v[:, ::32] = 2.0
    return v


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("which", ["w2", "x", "w1"])
def test_block_gradients_against_differences(cuda, p, which):
    import torch
    tokens, width, hidden, seed = 5, 40, 34, 11
    rng = np.random.default_rng(2)
    block = _block(tokens, width, hidden, p, torch.float32, seed)
    x, g = _on_grid(rng, tokens, width), _on_grid(rng, tokens, width)
    w2 = _on_grid(rng, width, hidden)
    # the inner matrix has to be on the grid too: hidden unit u sees input u, times 1
    w1 = np.zeros((hidden, width))
    w1[np.arange(hidden), np.arange(hidden)] = 1.0
    if which != "w2":
        # and so has its gradient, which W2 makes of G: unit u feeds output u, times 1
        w2 = w1.T.copy()

    def put(a):
        return torch.from_numpy(np.ascontiguousarray(a)).float().cuda()

    def loss(m):
        block.w1, block.w2 = put(m["w1"]), put(m["w2"])
        y = block.forward(put(m["x"]), step=1)
        return float((y.double() * put(g).double()).sum())

    at = {"x": x, "w1": w1, "w2": w2}
    loss(at)
    block.backward(put(g))
    grad = {"x": block.dx, "w1": block.dw1, "w2": block.dw2}[which].cpu().double().numpy()
    assert np.abs(grad).max() > 0

    def difference(i, j, step=0.5):
        up, down = ({k: v.copy() for k, v in at.items()} for _ in range(2))
        up[which][i, j] += step
        down[which][i, j] -= step
        return (loss(up) - loss(down)) / (2 * step)

    if which == "w1":
        # a unit's own weight, 1 +- 1/2, where its inputs are 0, 1 or 2 and the inner matrix stays on the grid
        places = [(u, u) for u in range(1, hidden) if u % 32 and np.all(np.isin(np.abs(x[:, u]), (0, 1, 2)))]
    else:
        # steps of 1/2 from magnitudes up to 1 1/2 stay on the grid; of an input that a unit sees, from
        # 1 and more, or -1 and less, so that its ReLU does not switch
        m = at[which]
        places = [(i, j) for i in range(1, m.shape[0]) for j in range(1, m.shape[1])
                  if i % 32 and j % 32 and abs(m[i, j]) <= 1.5
                  and not (which == "x" and j < hidden and abs(m[i, j]) < 1)]
        places = [places[k] for k in rng.choice(len(places), min(24, len(places)), replace=False)]
    assert len(places) >= 1
    for i, j in places:
        assert difference(i, j) == grad[i, j], (i, j)


def test_example_trains_and_serves(cuda):
    """The error falls below 0.6 of its start (0.36 / 1.51 in 32-bit arithmetic without
    quantisation), and single tokens give what a batch of them gives."""
    from mx4_feed_forward import main
    first, last, same = main(steps=200)
    assert last < 0.6 * first
    assert same
