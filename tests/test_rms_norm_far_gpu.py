"""GPU tests of sbx_rms_norm_grad where dy * w leaves what 32 bits hold and dy * w / rms does not; no eps.

dx: each of its terms is good to 8 * 2^-24 of its size (powers of two are exact; s, m and four products
are rounded), and the sum is rounded to its type once.  dw: a sum of `rows` products in 32 bits, off by at
most (rows + 8) 2^-24 of their magnitudes' sum."""
import numpy as np
import pytest

import layer_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 40, 700, 3000, 18000])
@pytest.mark.parametrize("scale,dy,w", [(-100, -80, -80), (126, 70, 60), (-140, -60, -45), (100, 50, 90), (-60, -90, -62),
                                        (0, -60, -60), (0, 60, 60)])
def test_products_past_32_bits(cuda, name, cols, scale, dy, w):
    import torch
    import sushiblas_amd as sbx
    dt, code = ref.types(name)
    rows, rng = 5, np.random.default_rng(cols)
    far = lambda shape, e: rng.uniform(0.5, 1.0, shape) * rng.choice([-1.0, 1.0], shape) * 2.0 ** e  # noqa: E731
    H, DY = ref.padded(cuda, far((rows, cols), scale), dt, 0), ref.padded(cuda, far((rows, cols), dy), dt, 0)
    W = ref.padded(cuda, far((1, cols), w), dt, 0)
    DX, DW = torch.full_like(H, 7.0), torch.full((cols,), 7.0, device=cuda)
    ws = torch.empty(sbx.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device=cuda)
    sbx.rms_norm_grad(code, rows, cols, H, cols, W, 0.0, DY, cols, DX, cols, DW=DW, workspace=ws)
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        dx, dw, size, sizew = ref.norm_grad(ref.f64(H), ref.f64(W)[0], 0.0, ref.f64(DY))
    got, gotw = ref.f64(DX), ref.f64(DW)
    if name == "bf16" and scale == -140:  # less than half of its least value, 2^-133: rows of zeros, whose gradients are NaN
        assert not ref.f64(H).any() and np.isnan(dx).all() and np.isnan(got).all() and np.isnan(gotw).all()
        return
    off = ref.HALF[name] * np.abs(dx) + 8 * 2.0 ** -24 * size
    assert (np.abs(got - dx) <= off * 1.01 + ref.TINY[name] * 1.01).all()
    assert (np.abs(gotw - dw) <= (rows + 8) * 2.0 ** -24 * sizew).all()
