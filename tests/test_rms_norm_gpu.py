"""GPU tests of sbx_rms_norm and sbx_mx8_dequantize against the plain implementation in 64 bits.

V is computed in 64 bits (its error, about (cols + 4) 2^-53 of it, does not count here), rounded
to 32 and, for Y, to its type: off by at most 2^-24 of it and half a step of the type.  H is the
sum in 32 bits rounded to its type, and MXFP8 the rounding of V in 32 bits: both bit for bit (a V
whose 64 bits lie within 2^-40 of a border of 32 may fall either way; the inputs have none, as
their being equal shows)."""
import numpy as np
import pytest

import layer_reference as ref

pytestmark = pytest.mark.gpu


def _near(got, want, name):
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    g, w = got[fine], want[fine]
    bound = (ref.HALF[name] * (1 + 2.0 ** -20) + (2.0 ** -24 if name != "f32" else 0.0)) * np.abs(w)
    assert (np.abs(g - w) <= bound + ref.TINY[name] * 1.01).all()


def _run(cuda, name, rows, cols, x=None, residual=True, eps=1e-6, pads=(0, 0, 0, 0, 0, 0), outs="hyq", w=None, alias="",
         stream=None, scale=1.0):
    """pads: of X, R, H, Y (elements), P (16 bytes), S (rows).  alias: "x", "r" (H, or Y without H, there)."""
    import torch
    import sushiblas_amd as sbx
    dt, code = ref.types(name)
    rng = np.random.default_rng(rows * 1009 + cols)
    x = rng.normal(size=(rows, cols)) * scale if x is None else x
    r = rng.normal(size=(rows, cols)) * 2 * scale if residual else None
    w = 1 + 0.1 * rng.normal(size=cols) if w is None else w
    X, R = ref.padded(cuda, x, dt, pads[0]), None if r is None else ref.padded(cuda, r, dt, pads[1])
    W = torch.from_numpy(w).to(dt).to(cuda)
    xf, rf = X.cpu()[:, :cols].float(), None if r is None else R.cpu()[:, :cols].float()
    h = (xf if r is None else xf + rf).to(dt)
    v = ref.norm(h.double().numpy(), ref.f64(W), eps)[0]
    H = torch.full((rows, cols + pads[2]), 7.0, dtype=dt, device=cuda) if "h" in outs else None
    Y = torch.full((rows, cols + pads[3]), 7.0, dtype=dt, device=cuda) if "y" in outs else None
    if alias:
        into = X if alias == "x" else R
        H, Y = (into, Y) if "h" in outs else (None, into)
    nb = -(-cols // 32)
    P = torch.full((rows, 32 * nb + 16 * pads[4]), 0xAB, dtype=torch.uint8, device=cuda) if "q" in outs else None
    S = torch.full((-(-nb // 8), 8 * (rows + pads[5])), 0xAB, dtype=torch.uint8, device=cuda) if "q" in outs else None
    ld = lambda t: 0 if t is None else t.shape[1]  # noqa: E731
    torch.cuda.synchronize()
    print("rms_norm", name, rows, cols, residual, eps, pads, outs, alias, flush=True)
    sbx.rms_norm(code, rows, cols, X, ld(X), W, eps, R=R, ldr=ld(R), H=H, ldh=ld(H), Y=Y, ldy=ld(Y), P=P, ldp=ld(P),
                 S=S, lds=ld(S), stream=stream)
    torch.cuda.synchronize()
    if H is not None:
        assert torch.equal(H.cpu()[:, :cols].view(torch.uint8), h.view(torch.uint8)) or np.array_equal(
            ref.f64(H)[:, :cols], h.double().numpy(), equal_nan=True)
    if Y is not None:
        _near(ref.f64(Y)[:, :cols], ref.rounded_to(v, dt) if not np.isfinite(v).all() else v, name)
    for t, given in ((H, 7.0), (Y, 7.0)):
        if t is not None and not alias:
            assert bool((t[:, cols:] == given).all())
    if P is not None:
        n, c = ref.quantize8(v)
        p, s = P.cpu().numpy(), S.cpu().numpy()
        np.testing.assert_array_equal(s, ref.codes(c, lds=8 * (rows + pads[5]), fill=0xAB))
        np.testing.assert_array_equal(p[:, :32 * nb], n.reshape(rows, 32 * nb))
        assert (p[:, 32 * nb:] == 0xAB).all()
        back = torch.full((rows, cols + 3), 7.0, dtype=dt, device=cuda)
        sbx.mx8_dequantize(code, rows, cols, P, ld(P), S, ld(S), back, cols + 3)
        want = ref.rounded_to(ref.values8(n, c, cols), dt)
        np.testing.assert_array_equal(ref.f64(back)[:, :cols], want)
        assert bool((back[:, cols:] == 7.0).all())
    return H, Y


COLS = [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, 257, 500, 511, 512, 513, 1000, 1023, 1024, 1025,
        2047, 2048, 2049, 4095, 4096, 4097, 5000, 8191, 8192, 8193, 12000, 16383, 16384, 16385, 20000, 33000]


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_columns(cuda, name, cols):
    _run(cuda, name, 3, cols)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (2, 70), (64, 5), (65, 64), (257, 300), (300, 1), (1000, 1024),
                                       (5000, 33), (70000, 8), (513, 2049), (40, 8200), (7, 17000)])
def test_rows(cuda, name, rows, cols):
    _run(cuda, name, rows, cols)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("pads", [(1, 2, 3, 5, 1, 1), (8, 0, 8, 0, 2, 0), (0, 8, 0, 16, 0, 3)])
@pytest.mark.parametrize("cols", [1, 40, 300, 1024, 4097, 16392])
def test_strides(cuda, name, pads, cols):
    _run(cuda, name, 5, cols, pads=pads)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("outs", ["h", "y", "q", "hy", "hq", "yq"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("cols", [72, 3000, 18000])
def test_outputs(cuda, name, outs, residual, cols):
    _run(cuda, name, 4, cols, residual=residual, outs=outs)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("outs,alias", [("hy", "x"), ("hyq", "r"), ("y", "x"), ("yq", "r")])
@pytest.mark.parametrize("cols", [33, 1000, 4096, 20000])
def test_in_place(cuda, name, outs, alias, cols):
    _run(cuda, name, 6, cols, outs=outs, alias=alias)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("cols", [40, 1025, 17000])
def test_values_that_are_not_finite(cuda, name, cols):
    x = np.random.default_rng(1).normal(size=(8, cols))
    x[0, 0], x[1, cols - 1], x[2, cols // 2] = np.nan, np.inf, -np.inf
    x[3] = 0.0
    x[4, :] = 0.0
    x[4, cols - 1] = 1.0
    _run(cuda, name, 8, cols, x=x, residual=False)
    _run(cuda, name, 8, cols, x=np.where(np.isfinite(x), x, 0.0), residual=False, eps=0.0)


@pytest.mark.parametrize("scale,eps", [(1e-3, 1e-6), (1e-30, 0.0), (1e18, 1e-6), (1.0, 1e30), (1e-38, 1e-60)])
def test_far_magnitudes(cuda, scale, eps):
    _run(cuda, "f32", 5, 300, scale=scale, eps=eps)
    _run(cuda, "bf16", 5, 300, scale=scale, eps=eps)


def test_borders_of_the_8_bit_form(cuda):
    """Rows of +-1 leave W itself: every tie between e4m3 values, what saturates, the smallest scales."""
    v = ref.e4m3_values()
    v = np.sort(v[np.isfinite(v) & (v >= 0)])
    ties = np.concatenate([v, (v[1:] + v[:-1]) / 2, [447.9, 448.0, 460.0, 480.0, 511.0]])
    w = np.zeros((len(ties), 32))
    w[:, 0], w[:, 1], w[:, 2] = 448.0, ties, -ties
    w[-5:, 0] = 500.0
    w = w.reshape(-1)
    for power in (0, -100, -130, 100):
        with np.errstate(under="ignore"):
            ww = np.float32(w * 2.0 ** power).astype(np.float64)
        x = np.where(np.arange(len(w)) % 3 == 0, -1.0, 1.0)[None].repeat(2, 0)
        _run(cuda, "f32", 2, len(w), x=x, residual=False, eps=0.0, w=ww)


def test_another_stream_and_replays(cuda):
    import torch
    import sushiblas_amd as sbx
    _run(cuda, "bf16", 50, 1000, stream=torch.cuda.Stream())
    x, r = torch.randn(37, 900, device=cuda).bfloat16(), torch.randn(37, 900, device=cuda).bfloat16()
    w = torch.ones(900, device=cuda).bfloat16()
    outs = [torch.empty_like(x) for _ in range(4)]

    def call(h, y):
        sbx.rms_norm(sbx.BF16, 37, 900, x, 900, w, 1e-6, R=r, ldr=900, H=h, ldh=900, Y=y, ldy=900)

    call(*outs[:2])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(*outs[2:])
    for i in range(3):
        x.copy_(torch.randn(37, 900, device=cuda))
        call(*outs[:2])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


def test_far_offsets(cuda):
    """Rows that lie past 2^32 bytes."""
    import torch
    import sushiblas_amd as sbx
    rows, cols, ld = 70, 40, (1 << 32) // 60
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of device memory")
    X = torch.empty((rows, ld), dtype=torch.bfloat16, device=cuda)
    Y = torch.empty((rows, ld), dtype=torch.bfloat16, device=cuda)
    X[:, :cols] = torch.randn(rows, cols, device=cuda)
    w = torch.ones(cols, device=cuda).bfloat16()
    sbx.rms_norm(sbx.BF16, rows, cols, X, ld, w, 1e-6, Y=Y, ldy=ld)
    _near(ref.f64(Y[:, :cols]), ref.norm(ref.f64(X[:, :cols]), np.ones(cols), 1e-6)[0], "bf16")
