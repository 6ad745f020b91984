"""GPU tests of sbx_mx4_moe against the plain implementation in 64 bits (layer_reference.moe, which
also bounds the error before the last rounding), and of a step of decoding: the norm, the
mixture, the norm to 8 bits and the layer that reads it.

Shares are rounded to 32 bits once.  Experts have to be the same: logits are sums in 64 bits, and
the inputs' differ by more than their rounding, or are equal."""
import numpy as np
import pytest

import layer_reference as ref
import mx4_reference as mx4

pytestmark = pytest.mark.gpu

ROUNDED = {"f32": 2.0 ** -22, "bf16": 2.0 ** -15, "f16": 2.0 ** -15}  # of activations: cut to 24 or 16 bits


class Mixture:
    def __init__(self, cuda, name, width, hidden, experts, seed=1, pads=(0, 0, 0, 0, 0), same=()):
        """pads: of W1, W2 (blocks), S1, S2 (rows), WR (elements); same: experts with one router row."""
        import torch
        self.name, self.width, self.hidden, self.experts, self.cuda = name, width, hidden, experts, cuda
        self.dt, self.code = ref.types(name)
        rng = np.random.default_rng(seed + width * 7 + hidden)
        # elements are about 2.5 in size: scales that make a result of the size of its input
        c1, c2 = 126 - int(np.log2(width) / 2), 126 - int(np.log2(hidden) / 2)
        n1, s1, w1 = ref.random_mx4(rng, experts * 2 * hidden, width, c1 - 1, c1 + 1)
        n2, s2, w2 = ref.random_mx4(rng, experts * width, hidden, c2 - 1, c2 + 1)
        self.w1, self.w2 = w1.reshape(experts, 2 * hidden, width), w2.reshape(experts, width, hidden)
        self.W1, self.S1 = ref.packed(cuda, n1, s1, pads[0], pads[2])
        self.W2, self.S2 = ref.packed(cuda, n2, s2, pads[1], pads[3])
        wr = rng.normal(size=(experts, width)) * width ** -0.5
        for e in same:
            wr[e] = wr[same[0]]
        self.WR = ref.padded(cuda, wr, self.dt, pads[4])
        self.wr = ref.f64(self.WR)[:, :width]
        torch.cuda.synchronize()

    def call(self, X, Y, topk, normalize, chosen=None, weights=None, ws=None, stream=None, ldx=None, ldy=None):
        import torch
        import sushiblas_amd as sbx
        sizes = (X.shape[0], self.width, self.hidden, self.experts, topk)
        need = sbx.mx4_moe_workspace(*sizes)
        if ws is None:
            ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=self.cuda)
        sbx.mx4_moe(self.code, *sizes, X, X.stride(0), self.WR, self.WR.shape[1], self.W1, self.W1.shape[1], self.S1,
                    self.S1.shape[1], self.W2, self.W2.shape[1], self.S2, self.S2.shape[1], Y, Y.stride(0),
                    normalize=normalize, chosen=chosen, weights=weights, workspace=ws, workspace_bytes=need,
                    stream=stream)

    def check(self, x, topk, normalize=True, pads=(0, 0), stream=None, outs=True):
        import torch
        tokens = x.shape[0]
        X = ref.padded(self.cuda, x, self.dt, pads[0])
        Y = torch.full((tokens, self.width + pads[1]), 7.0, dtype=self.dt, device=self.cuda)
        chosen = torch.full((tokens * topk + 1,), -7, dtype=torch.int32, device=self.cuda) if outs else None
        weights = torch.full((tokens * topk + 1,), 7.0, device=self.cuda) if outs else None
        torch.cuda.synchronize()
        print("mx4_moe", self.name, tokens, self.width, self.hidden, self.experts, topk, normalize, pads, flush=True)
        self.call(X, Y, topk, normalize, chosen, weights, stream=stream)
        torch.cuda.synchronize()
        y, off, order, p = ref.moe(ref.f64(X)[:, :self.width], self.wr, self.w1, self.w2, topk, normalize,
                                   ROUNDED[self.name])
        if outs:
            c, w = chosen.cpu().numpy(), ref.f64(weights)
            np.testing.assert_array_equal(c[:-1].reshape(tokens, topk), order)
            got = w[:-1].reshape(tokens, topk)
            np.testing.assert_array_equal(np.isnan(got), np.isnan(p))
            assert (np.abs(got - p) <= 2.0 ** -23 * p + 2.0 ** -149)[~np.isnan(p)].all()
            assert c[-1] == -7 and w[-1] == 7.0
        got = ref.f64(Y)
        assert (got[:, self.width:] == 7.0).all()
        got = got[:, :self.width]
        np.testing.assert_array_equal(np.isnan(got), np.isnan(y))
        fine = np.isfinite(y)
        assert (np.abs(got - y) <= off + ref.HALF[self.name] * (np.abs(y) + off) + ref.TINY[self.name])[fine].all()
        # and far nearer than the bound on the whole
        if fine.all() and y.size >= 64:
            assert np.linalg.norm(got - y) <= (ref.HALF[self.name] + 2.0 ** -14 * (self.name != "f32") + 4e-6) * np.linalg.norm(y)
        return Y


def _x(tokens, width, seed=0):
    return np.random.default_rng(tokens * 31 + width + seed).normal(size=(tokens, width))


SIZES = [(1, 32, 32, 2, 1), (1, 1, 1, 1, 1), (3, 40, 70, 5, 2), (1, 256, 256, 8, 2), (2, 300, 100, 9, 3), (1, 1024, 512, 64, 8),
         (7, 1000, 700, 9, 2), (16, 96, 64, 4, 4), (33, 130, 72, 3, 2), (17, 512, 257, 16, 4), (64, 200, 96, 12, 3),
         (40, 64, 40, 1, 1), (5, 2049, 33, 7, 1), (4, 65, 2100, 6, 2), (100, 48, 31, 20, 5), (256, 33, 34, 5, 2),
         (20, 100, 100, 300, 16), (3, 64, 64, 512, 8)]


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("tokens,width,hidden,experts,topk", SIZES)
def test_sizes(cuda, name, tokens, width, hidden, experts, topk):
    Mixture(cuda, name, width, hidden, experts).check(_x(tokens, width), topk)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("pads,xp", [((1, 1, 1, 1, 1), (1, 3)), ((0, 3, 5, 0, 8), (8, 8)), ((2, 0, 0, 2, 0), (0, 1))])
def test_strides_and_shares(cuda, name, normalize, pads, xp):
    for tokens, width, hidden, experts, topk in ((1, 300, 200, 6, 2), (9, 72, 135, 4, 3)):
        Mixture(cuda, name, width, hidden, experts, pads=pads).check(_x(tokens, width), topk, normalize, xp)


@pytest.mark.parametrize("name", ref.TYPES)
def test_equal_logits_go_by_index(cuda, name):
    m = Mixture(cuda, name, 96, 64, 8, same=(1, 3, 4, 6))
    m.check(_x(12, 96), 3)
    m.check(np.zeros((2, 96)), 4, False)  # all equal


def test_all_tokens_choose_the_same(cuda):
    """One expert gets every token: several tiles of it."""
    m = Mixture(cuda, "bf16", 128, 96, 6)
    x = _x(1, 128).repeat(70, 0) * (1 + np.arange(70) % 3)[:, None]
    m.check(x, 2)


@pytest.mark.parametrize("name", ref.TYPES)
def test_values_that_are_not_finite(cuda, name):
    m = Mixture(cuda, name, 70, 40, 5)
    x = _x(6, 70)
    x[1, 3], x[4, 69] = np.nan, np.nan
    m.check(x, 2)
    m.check(x, 5, False)


@pytest.mark.parametrize("name", ref.TYPES)
def test_infinite_values_stay_with_their_token(cuda, name):
    import torch
    m = Mixture(cuda, name, 70, 40, 5)
    x = _x(6, 70)
    want = m.check(x, 2)
    x[2, 0] = np.inf
    X, Y = ref.padded(cuda, x, m.dt, 0), torch.empty_like(want)
    chosen = torch.full((6, 2), -1, dtype=torch.int32, device=cuda)
    m.call(X, Y, 2, True, chosen)
    assert not bool(torch.isfinite(Y[2]).any()) and bool(((chosen >= 0) & (chosen < 5)).all())
    others = [0, 1, 3, 4, 5]
    assert torch.equal(Y[others], want[others])


def test_without_the_choices(cuda):
    Mixture(cuda, "f16", 100, 60, 7).check(_x(3, 100), 2, outs=False)


def test_same_bits_again_streams_workspaces_and_replays(cuda):
    import torch
    import sushiblas_amd as sbx
    m = Mixture(cuda, "bf16", 512, 256, 16)
    x = torch.randn(11, 512, device=cuda).bfloat16()
    sizes = (11, 512, 256, 16, 4)
    ys = [torch.empty_like(x) for _ in range(3)]
    ws = [torch.full((sbx.mx4_moe_workspace(*sizes),), 0xFF, dtype=torch.uint8, device=cuda) for _ in range(2)]
    m.call(x, ys[0], 4, True, ws=ws[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.call(x, ys[1], 4, True, ws=ws[1])
    side = torch.cuda.Stream()
    for _ in range(3):
        x.copy_(torch.randn(11, 512, device=cuda))
        m.call(x, ys[0], 4, True, ws=ws[0])
        g.replay()
        torch.cuda.synchronize()
        m.call(x, ys[2], 4, True, ws=ws[0], stream=side)
        torch.cuda.synchronize()
        assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


@pytest.mark.parametrize("tokens", [1, 5, 90])
def test_in_place(cuda, tokens):
    import torch
    m = Mixture(cuda, "bf16", 300, 130, 9)
    x = torch.randn(tokens, 310, device=cuda).bfloat16()
    y, was = x.clone(), x.clone()
    m.call(x[:, :300], y[:, :300], 3, False)
    m.call(x[:, :300], x[:, :300], 3, False)
    assert torch.equal(x, y) and torch.equal(x[:, 300:], was[:, 300:])


def test_two_at_once(cuda):
    """Calls on two streams, a workspace each, of the same weights."""
    import torch
    import sushiblas_amd as sbx
    m = Mixture(cuda, "f16", 1024, 512, 16)
    streams, xs, ys = [torch.cuda.Stream() for _ in range(2)], [], []
    for tokens in (3, 40):
        xs.append(torch.randn(tokens, 1024, device=cuda).half())
        ys.append([torch.empty_like(xs[-1]) for _ in range(9)])
        m.call(xs[-1], ys[-1][0], 4, True)
    ws = [torch.empty(sbx.mx4_moe_workspace(x.shape[0], 1024, 512, 16, 4), dtype=torch.uint8, device=cuda) for x in xs]
    torch.cuda.synchronize()
    for i in range(1, 9):
        for x, y, s, w in zip(xs, ys, streams, ws):
            m.call(x, y[i], 4, True, ws=w, stream=s)
    torch.cuda.synchronize()
    for y in ys:
        assert all(torch.equal(y[0], other) for other in y[1:])


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("tokens", [1, 6])
def test_a_step_of_decoding(cuda, name, tokens):
    """x + r -> norm -> mixture -> + residual -> norm to 8 bits -> a layer, each on what the call before
    it wrote; each result is checked against the formula on that."""
    import torch
    import sushiblas_amd as sbx
    width, out = 512, 1000
    dt, code = ref.types(name)
    m = Mixture(cuda, name, width, 256, 8)
    rng = np.random.default_rng(9)
    x, r = (ref.padded(cuda, rng.normal(size=(tokens, width)), dt, 0) for _ in range(2))
    w = torch.from_numpy(1 + 0.1 * rng.normal(size=width)).to(dt).to(cuda)
    wn, wc, wl = ref.random_mx4(rng, out, width, 121, 123)
    B, SB = ref.packed(cuda, wn, wc)
    new = lambda n: torch.empty((tokens, n), dtype=dt, device=cuda)  # noqa: E731
    h, y, z, h2, logits = new(width), new(width), new(width), new(width), new(out)
    P, S = (torch.empty(s, dtype=torch.uint8, device=cuda) for s in sbx.mx8_shapes(tokens, width))
    sbx.rms_norm(code, tokens, width, x, width, w, 1e-6, R=r, ldr=width, H=h, ldh=width, Y=y, ldy=width)
    m.call(y, z, 2, True)
    sbx.rms_norm(code, tokens, width, z, width, w, 1e-6, R=h, ldr=width, H=h2, ldh=width, P=P, ldp=P.stride(0), S=S,
                 lds=S.stride(0))
    sbx.mx4_linear(code, tokens, out, width, 1.0, P, P.stride(0), B, B.stride(0), SB, SB.stride(0), 0.0, logits, out,
                   SX=S, ldsx=S.stride(0))
    torch.cuda.synchronize()
    half = ref.HALF[name]
    v = ref.norm(ref.f64(h), ref.f64(w), 1e-6)[0]
    assert (np.abs(ref.f64(y) - v) <= (half + 2.0 ** -23) * np.abs(v)).all()
    want, off, _, _ = ref.moe(ref.f64(y), m.wr, m.w1, m.w2, 2, True, ROUNDED[name])
    assert (np.abs(ref.f64(z) - want) <= off + half * (np.abs(want) + off)).all()
    n, c = ref.quantize8(ref.norm(ref.f64(h2), ref.f64(w), 1e-6)[0])
    a = ref.values8(n, c, width)
    want, bound = a @ wl.T, (width + 4) * 2.0 ** -24 * (np.abs(a) @ np.abs(wl).T)
    assert (np.abs(ref.f64(logits) - want) <= bound + half * (np.abs(want) + bound)).all()
