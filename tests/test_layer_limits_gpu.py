"""GPU tests of the norm, the few-token layer and the mixture at sizes whose offsets pass 32 bits, or
whose workgroups pass what one dimension of a launch takes: long rows, tall weights, far leading
dimensions.  Values repeat a short table's, or are compared on the device."""
import numpy as np
import pytest

import layer_reference as ref
import mx4_reference as mx4

pytestmark = pytest.mark.gpu


def _room(gib):
    import torch
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


def test_norm_and_gradient_of_a_long_row(cuda):
    """One row of 2^28 + 5 columns: values of a period, so that sums are known and results repeat."""
    import torch
    import sushiblas_amd as sbx
    _room(30)
    cols, period = (1 << 28) + 5, 1 << 12
    rng = np.random.default_rng(1)
    whole = cols // period
    table = {n: torch.from_numpy(rng.normal(size=period)).bfloat16() for n in ("h", "w", "dy")}
    h, w, dy = (table[n].to(cuda).repeat(whole + 1)[:cols].contiguous() for n in ("h", "w", "dy"))
    f = {n: t.double().numpy() for n, t in table.items()}
    full = lambda a: (a.sum() * whole + a[:cols - whole * period].sum()) / cols  # noqa: E731
    s = 1 / np.sqrt(full(f["h"] ** 2) + 1e-6)
    along = full(f["dy"] * f["w"] * f["h"])

    def repeats(t, want, bound):
        """t's values are the table's, over and over, to `bound`."""
        want, bound = torch.from_numpy(want).to(cuda), torch.from_numpy(bound).to(cuda)
        for at in range(0, whole, 1 << 12):
            part = t[at * period:min(at + (1 << 12), whole) * period].double().reshape(-1, period)
            assert bool(((part - want).abs() <= bound).all())
        end = cols - whole * period
        assert bool(((t[whole * period:].double() - want[:end]).abs() <= bound[:end]).all())

    y = torch.empty(cols, dtype=torch.bfloat16, device=cuda)
    print("rms_norm 1 x", cols, flush=True)
    sbx.rms_norm(sbx.BF16, 1, cols, h, cols, w, 1e-6, Y=y, ldy=cols)
    v = f["h"] * s * f["w"]
    repeats(y, v, (2.0 ** -8 + 2.0 ** -22) * np.abs(v))
    dx, dw = y, torch.empty(cols, device=cuda)
    ws = torch.empty(sbx.rms_norm_grad_workspace(1, cols), dtype=torch.uint8, device=cuda)
    print("rms_norm_grad 1 x", cols, flush=True)
    sbx.rms_norm_grad(sbx.BF16, 1, cols, h, cols, w, 1e-6, dy, cols, dx, cols, DW=dw, workspace=ws)
    g = f["dy"] * f["w"]
    want = s * g - f["h"] * s ** 3 * along
    size = np.abs(s * g) + np.abs(f["h"]) * s ** 3 * full(np.abs(g * f["h"]))
    repeats(dx, want, 2.0 ** -8 * np.abs(want) + 9 * 2.0 ** -24 * size)
    want = s * f["dy"] * f["h"]
    repeats(dw, want, 9 * 2.0 ** -24 * np.abs(want))


@pytest.mark.parametrize("mx8", [False, True])
def test_linear_of_a_tall_weight(cuda, mx8):
    """2^28 + 7 results of 32 terms, their rows a table's over and over."""
    import torch
    import sushiblas_amd as sbx
    _room(20)
    n, period = (1 << 28) + 7, 1 << 12
    rng = np.random.default_rng(2)
    wn, wc, w = ref.random_mx4(rng, period, 32, 126, 129)
    P, S = mx4.pack(wn, wc)
    whole = n // period
    B = torch.from_numpy(P).to(cuda).repeat(whole + 1, 1)[:n].contiguous()
    SB = torch.from_numpy(S.reshape(period, 8)).to(cuda).repeat(whole + 1, 1)[:n].contiguous()
    x = rng.integers(-8, 9, (1, 32)).astype(np.float64)
    y = torch.empty(n, device=cuda)
    print("mx4_linear 1 x", n, "x 32", mx8, flush=True)
    if mx8:
        xn, xc = ref.quantize8(x)
        X, SX = torch.from_numpy(xn.reshape(1, 32)).to(cuda), torch.from_numpy(ref.codes(xc)).to(cuda)
        x = ref.values8(xn, xc, 32)
        sbx.mx4_linear(sbx.F32, 1, n, 32, 1.0, X, 32, B, 16, SB, 8 * n, 0.0, y, n, SX=SX, ldsx=8)
    else:
        sbx.mx4_linear(sbx.F32, 1, n, 32, 1.0, torch.from_numpy(x).float().to(cuda), 32, B, 16, SB, 8 * n, 0.0, y, n)
    want = torch.from_numpy((x @ w.T)[0]).float().to(cuda)  # (exact in 32 bits)
    for at in range(0, whole, 1 << 12):
        assert bool((y[at * period:min(at + (1 << 12), whole) * period].reshape(-1, period) == want).all())
    assert torch.equal(y[whole * period:], want[:n - whole * period])


def test_linear_with_far_leading_dimensions(cuda):
    """Rows of the weight 2^23 - 16 bytes apart, of X 2^26: the largest that are taken."""
    import torch
    import sushiblas_amd as sbx
    _room(8)
    rng = np.random.default_rng(3)
    m, n, k, ldb, ldx = 17, 70, 300, (1 << 23) - 16, 1 << 25
    wn, wc, w = ref.random_mx4(rng, n, k, 126, 129)
    P, S = mx4.pack(wn, wc)
    B = torch.zeros((n, ldb), dtype=torch.uint8, device=cuda)
    B[:, :P.shape[1]] = torch.from_numpy(P).to(cuda)
    SB = torch.from_numpy(S).to(cuda)
    x = rng.integers(-8, 9, (m, k)).astype(np.float64)
    X = torch.zeros((m, ldx), dtype=torch.bfloat16, device=cuda)
    X[:, :k] = torch.from_numpy(x).bfloat16().to(cuda)
    y = torch.empty((m, n), dtype=torch.bfloat16, device=cuda)
    print("mx4_linear far", flush=True)
    sbx.mx4_linear(sbx.BF16, m, n, k, 1.0, X, ldx, B, ldb, SB, SB.shape[1], 0.0, y, n)
    np.testing.assert_array_equal(ref.f64(y), ref.rounded_to(x @ w.T, torch.bfloat16))
    xn, xc = ref.quantize8(x)
    X8 = torch.zeros((m, 1 << 26), dtype=torch.uint8, device=cuda)
    X8[:, :xc.shape[1] * 32] = torch.from_numpy(xn.reshape(m, -1)).to(cuda)
    SX = torch.from_numpy(ref.codes(xc)).to(cuda)
    sbx.mx4_linear(sbx.BF16, m, n, k, 1.0, X8, 1 << 26, B, ldb, SB, SB.shape[1], 0.0, y, n, SX=SX, ldsx=8 * m)
    np.testing.assert_array_equal(ref.f64(y), ref.rounded_to(ref.values8(xn, xc, k) @ w.T, torch.bfloat16))


@pytest.mark.parametrize("tokens", [1, 3, 70])
def test_mixture_past_32_bits(cuda, tokens):
    """Experts' weights in rows 2^21 bytes apart, 5 and 8 GB in all, tokens in rows just below 2^23."""
    import torch
    import sushiblas_amd as sbx
    _room(24)
    rng = np.random.default_rng(4)
    width, hidden, experts, topk, ld, ldx = 48, 40, 60, 4, 1 << 21, (1 << 22) - 8
    n1, c1, w1 = ref.random_mx4(rng, experts * 2 * hidden, width, 122, 125)
    n2, c2, w2 = ref.random_mx4(rng, experts * width, hidden, 122, 125)

    def far(n, c):
        P, S = mx4.pack(n, c)
        t = torch.zeros((P.shape[0], ld), dtype=torch.uint8, device=cuda)
        t[:, :P.shape[1]] = torch.from_numpy(P).to(cuda)
        return t, torch.from_numpy(S).to(cuda)

    (W1, S1), (W2, S2) = far(n1, c1), far(n2, c2)
    WR = torch.from_numpy(rng.normal(size=(experts, width)) * width ** -0.5).bfloat16().to(cuda)
    X = torch.zeros((tokens, ldx), dtype=torch.bfloat16, device=cuda)
    X[:, :width] = torch.from_numpy(rng.normal(size=(tokens, width))).bfloat16().to(cuda)
    Y = torch.empty((tokens, width), dtype=torch.bfloat16, device=cuda)
    sizes = (tokens, width, hidden, experts, topk)
    ws = torch.empty(sbx.mx4_moe_workspace(*sizes), dtype=torch.uint8, device=cuda)
    print("mx4_moe far", tokens, flush=True)
    sbx.mx4_moe(sbx.BF16, *sizes, X, ldx, WR, width, W1, ld, S1, S1.shape[1], W2, ld, S2, S2.shape[1], Y, width,
                workspace=ws)
    y, off, _, _ = ref.moe(ref.f64(X[:, :width]), ref.f64(WR), w1.reshape(experts, 2 * hidden, width),
                           w2.reshape(experts, width, hidden), topk, True, 2.0 ** -15)
    assert (np.abs(ref.f64(Y) - y) <= off + 2.0 ** -8 * (np.abs(y) + off)).all()


def test_mixture_of_wide_tokens(cuda):
    """The widest hidden layer and tokens that are taken, one expert."""
    import torch
    import sushiblas_amd as sbx
    _room(8)
    rng = np.random.default_rng(5)
    for width, hidden in ((40, 1 << 18), (1 << 18, 40)):
        n1, c1, w1 = ref.random_mx4(rng, 2 * hidden, width, 117, 118)
        n2, c2, w2 = ref.random_mx4(rng, width, hidden, 117, 118)
        W1, S1 = ref.packed(cuda, n1, c1)
        W2, S2 = ref.packed(cuda, n2, c2)
        for tokens in (1, 2):
            x = torch.from_numpy(rng.normal(size=(tokens, width))).bfloat16()
            X, WR = x.to(cuda), torch.zeros((1, width), dtype=torch.bfloat16, device=cuda)
            Y = torch.empty_like(X)
            sizes = (tokens, width, hidden, 1, 1)
            ws = torch.empty(sbx.mx4_moe_workspace(*sizes), dtype=torch.uint8, device=cuda)
            print("mx4_moe", sizes, flush=True)
            sbx.mx4_moe(sbx.BF16, *sizes, X, width, WR, width, W1, W1.shape[1], S1, S1.shape[1], W2, W2.shape[1], S2,
                        S2.shape[1], Y, width, workspace=ws)
            y, off, _, _ = ref.moe(x.double().numpy(), np.zeros((1, width)), w1[None], w2[None], 1, True, 2.0 ** -15)
            assert (np.abs(ref.f64(Y) - y) <= off + 2.0 ** -8 * (np.abs(y) + off)).all()
