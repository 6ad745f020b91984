"""GPU tests of sbx_rms_norm_grad against the formula in 64 bits, and against differences.

dx: each of its terms is good to 8 * 2^-24 of its size (a few operations in 32 bits, or in 64),
and the sum is rounded to its type once.  dw: a sum of `rows` products in 32 bits, off by at most
(rows + 8) 2^-24 of their magnitudes' sum."""
import numpy as np
import pytest

import layer_reference as ref

pytestmark = pytest.mark.gpu


def _run(cuda, name, rows, cols, dr=True, dw=True, pads=(0, 0, 0, 0), alias="", eps=1e-6, h=None, stream=None,
         dy=1.0):
    import torch
    import sushiblas_amd as sbx
    dt, code = ref.types(name)
    rng = np.random.default_rng(rows * 1013 + cols)
    h = rng.normal(size=(rows, cols)) if h is None else h
    H = ref.padded(cuda, h, dt, pads[0])
    DY = ref.padded(cuda, rng.normal(size=(rows, cols)) * dy, dt, pads[1])
    DR = ref.padded(cuda, rng.normal(size=(rows, cols)), dt, pads[2]) if dr else None
    W = torch.from_numpy(1 + 0.1 * rng.normal(size=cols)).to(dt).to(cuda)
    with np.errstate(invalid="ignore"):
        want, wantw, size, sizew = ref.norm_grad(ref.f64(H)[:, :cols], ref.f64(W), eps, ref.f64(DY)[:, :cols],
                                                 ref.f64(DR)[:, :cols] if dr else None)
    DX = {"": torch.full((rows, cols + pads[3]), 7.0, dtype=dt, device=cuda), "dy": DY, "dr": DR}[alias]
    DW = torch.full((cols + 1,), 7.0, device=cuda) if dw else None
    need = sbx.rms_norm_grad_workspace(rows, cols)
    ws = torch.full((need + 16,), 0xFF, dtype=torch.uint8, device=cuda) if dw else None  # NaN
    torch.cuda.synchronize()
    print("rms_norm_grad", name, rows, cols, dr, dw, pads, alias, flush=True)
    sbx.rms_norm_grad(code, rows, cols, H, H.shape[1], W, eps, DY, DY.shape[1], DX, DX.shape[1], DW=DW, DR=DR,
                      lddr=DR.shape[1] if dr else 0, workspace=ws, workspace_bytes=need if dw else 0, stream=stream)
    torch.cuda.synchronize()
    got = ref.f64(DX)[:, :cols]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = np.isfinite(want)
    off = np.abs(got - want)[ok]
    assert (off <= (ref.HALF[name] * np.abs(want) + 8 * 2.0 ** -24 * size)[ok] * 1.01 + ref.TINY[name] * 1.01).all()
    if not alias:
        assert bool((DX[:, cols:] == 7.0).all())
    if dw:
        gotw = ref.f64(DW)
        assert gotw[cols] == 7.0 and bool((ws[need:] == 0xFF).all())
        np.testing.assert_array_equal(np.isnan(gotw[:cols]), np.isnan(wantw))
        ok = np.isfinite(wantw)
        assert (np.abs(gotw[:cols] - wantw)[ok] <= ((rows + 8) * 2.0 ** -24 * sizew)[ok]).all()
    return DX, DW


COLS = [1, 3, 8, 31, 64, 65, 130, 256, 500, 512, 513, 1000, 1024, 2047, 2048, 2056, 4096, 5001, 8192, 9000, 16384, 16400,
        33000]


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_columns(cuda, name, cols):
    _run(cuda, name, 5, cols)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2048), (255, 40), (256, 1024), (257, 1024), (600, 2100), (3000, 100),
                                       (20000, 17), (2000, 1), (259, 8208), (300, 17000)])
def test_rows(cuda, name, rows, cols):
    _run(cuda, name, rows, cols)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("dr,dw,pads,alias", [(False, True, (1, 2, 0, 3), ""), (True, False, (3, 1, 2, 5), ""),
                                              (False, False, (8, 8, 0, 8), ""), (True, True, (0, 8, 8, 0), "dy"),
                                              (True, True, (2, 0, 1, 0), "dr"), (False, True, (0, 0, 0, 0), "dy")])
@pytest.mark.parametrize("cols", [30, 1100, 4096, 17000])
def test_forms(cuda, name, dr, dw, pads, alias, cols):
    _run(cuda, name, 300, cols, dr, dw, pads, alias)


@pytest.mark.parametrize("cols", [40, 3000, 18000])
def test_values_that_are_not_finite(cuda, cols):
    h = np.random.default_rng(1).normal(size=(6, cols))
    h[0, 0], h[2, cols - 1] = np.nan, np.inf
    h[3] = 0.0
    _run(cuda, "f32", 6, cols, h=h, dw=False)
    _run(cuda, "bf16", 6, cols, h=h, dw=False)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 40, 3000, 18000])
@pytest.mark.parametrize("scale,dy", [(-130, -20), (-100, -20), (-60, 0), (70, 0), (126, 60)])
def test_far_magnitudes(cuda, name, cols, scale, dy):
    """1 / rms past what 32 bits hold, below their normal numbers, and between; no eps."""
    h = np.random.default_rng(cols).uniform(0.5, 1.0, size=(5, cols)) * 2.0 ** scale
    h[:, ::2] *= -1
    _run(cuda, name, 5, cols, dr=False, eps=0.0, h=h, dy=2.0 ** dy)


def test_no_rows(cuda):
    import torch
    import sushiblas_amd as sbx
    dw = torch.full((70,), 7.0, device=cuda)
    sbx.rms_norm_grad(sbx.F32, 0, 69, None, 69, None, 1e-6, None, 69, None, 69, DW=dw)
    assert bool((dw[:69] == 0).all()) and float(dw[69]) == 7.0


def test_same_bits_again_other_streams_and_replays(cuda):
    import torch
    import sushiblas_amd as sbx
    a = _run(cuda, "bf16", 700, 1500)
    b = _run(cuda, "bf16", 700, 1500, stream=torch.cuda.Stream())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    rows, cols = 300, 700
    h, dy = torch.randn(rows, cols, device=cuda), torch.randn(rows, cols, device=cuda)
    w, ws = torch.ones(cols, device=cuda), torch.empty(sbx.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device=cuda)
    dx, dw = [torch.empty_like(h) for _ in range(2)], [torch.empty(cols, device=cuda) for _ in range(2)]

    def call(i):
        sbx.rms_norm_grad(sbx.F32, rows, cols, h, cols, w, 1e-6, dy, cols, dx[i], cols, DW=dw[i], workspace=ws)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(1)
    for _ in range(3):
        dy.copy_(torch.randn(rows, cols, device=cuda))
        call(0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx[0], dx[1]) and torch.equal(dw[0], dw[1])


def test_against_differences(cuda):
    """The library's gradient in 32 bits against differences of the norm in 64: off by d^2 and rounding."""
    import torch
    dx, dw = _run(cuda, "f32", 2, 9, dr=False)
    rng = np.random.default_rng(2 * 1013 + 9)
    f32 = lambda a: a.astype(np.float32).astype(np.float64)  # noqa: E731
    h, dy, w = f32(rng.normal(size=(2, 9))), f32(rng.normal(size=(2, 9))), f32(1 + 0.1 * rng.normal(size=9))
    loss = lambda h, w: (ref.norm(h, w, 1e-6)[0] * dy).sum()  # noqa: E731
    d = 1e-5
    for i in np.ndindex(2, 9):
        e = np.zeros((2, 9))
        e[i] = d
        assert abs((loss(h + e, w) - loss(h - e, w)) / (2 * d) - float(dx[i])) < 1e-5
    for i in range(9):
        e = np.zeros(9)
        e[i] = d
        assert abs((loss(h, w + e) - loss(h, w - e)) / (2 * d) - float(dw[i])) < 1e-5
    del torch
