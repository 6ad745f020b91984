"""GPU tests of sbx_dropout against the plain implementation (mx4_reference).

The operator's arithmetic is one multiplication, in 32 bits (64 for F64) with
one rounding to the type, and a mask: results have to be equal, bit for bit.
"""
import numpy as np
import pytest

import mx4_reference as ref

pytestmark = pytest.mark.gpu

SEED = 0x1234567890ABCDEF
TYPES = ["f32", "f64", "bf16", "f16"]


def _types(name):
    import torch
    import sushiblas_amd as sbx
    return {"f32": (torch.float32, sbx.F32), "f64": (torch.float64, sbx.F64),
            "bf16": (torch.bfloat16, sbx.BF16), "f16": (torch.float16, sbx.F16)}[name]


def _np(t):
    """A host copy in a type numpy has (bf16 and f16 values as float32)."""
    import torch
    t = t.cpu()
    return (t if t.dtype in (torch.float32, torch.float64) else t.float()).numpy()


def _rounded(y, dt):
    import torch
    return torch.from_numpy(np.ascontiguousarray(y)).to(dt)


def _bits(t):
    import torch
    return t.contiguous().view({8: torch.int64, 4: torch.int32, 2: torch.int16}[t.element_size()])


def _run(cuda, name, rows, cols, p, gate, pads=(0, 0, 0), sid=5, stream=None):
    import torch
    import sushiblas_amd as sbx
    dt, code = _types(name)
    gen = torch.Generator().manual_seed(rows * 7 + cols)
    x = torch.randn((rows, cols + pads[0]), generator=gen, dtype=torch.float64).to(dt)
    g = torch.randn((rows, cols + pads[1]), generator=gen, dtype=torch.float64).to(dt)
    y = torch.full((rows, cols + pads[2]), 7.0, dtype=dt)
    dx, dg, dy = x.to(cuda), g.to(cuda), y.to(cuda)
    torch.cuda.synchronize()
    print("dropout", name, rows, cols, p, gate, pads, flush=True)
    sbx.dropout(code, rows, cols, dx, cols + pads[0], dy, cols + pads[2], p, SEED, sid,
                gate=dg if gate else None, ldg=cols + pads[1], stream=stream)
    torch.cuda.synchronize()
    want = ref.dropped(_np(x[:, :cols]), p, SEED, sid, _np(g[:, :cols]) if gate else None)
    got = dy.cpu()
    assert torch.equal(_bits(got[:, :cols]), _bits(_rounded(want, dt)))
    assert torch.equal(got[:, cols:], y[:, cols:])  # what is between rows stays
    assert torch.equal(_bits(dx.cpu()), _bits(x))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 8), (5, 9), (300, 1), (17, 250), (64, 2048),
                                       (129, 2051), (2, 20000)])
def test_dropout_sizes(cuda, name, rows, cols):
    _run(cuda, name, rows, cols, 0.1, False)
    _run(cuda, name, rows, cols, 0.5, True)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("pads", [(1, 0, 0), (0, 3, 1), (8, 8, 8), (5, 1, 2)])
def test_dropout_leading_dimensions(cuda, name, pads):
    _run(cuda, name, 37, 121, 0.3, True, pads)


@pytest.mark.parametrize("p", [0.0, 1e-7, 0.25, 0.99999, 1.0])
def test_dropout_rates(cuda, p):
    """p rounds to a multiple of 2^-16: nothing, all but a few and everything dropped."""
    _run(cuda, "f32", 65, 300, p, False)
    _run(cuda, "bf16", 65, 300, p, True)


@pytest.mark.parametrize("name", TYPES)
def test_dropout_in_place_and_twice(cuda, name):
    """Y may be X; the same call gives the same mask, another stream_id or seed another."""
    import torch
    import sushiblas_amd as sbx
    dt, code = _types(name)
    x = torch.ones((50, 70), dtype=dt, device=cuda)
    a, b, c, d = (torch.empty_like(x) for _ in range(4))
    sbx.dropout(code, 50, 70, x, 70, a, 70, 0.5, 9, 1)
    sbx.dropout(code, 50, 70, x, 70, b, 70, 0.5, 9, 2)
    sbx.dropout(code, 50, 70, x, 70, c, 70, 0.5, 10, 1)
    sbx.dropout(code, 50, 70, x, 70, d, 70, 0.5, 9 + (1 << 32), 1)
    sbx.dropout(code, 50, 70, x, 70, x, 70, 0.5, 9, 1)
    assert torch.equal(x, a)
    assert not torch.equal(a, b) and not torch.equal(a, c) and not torch.equal(a, d)


def test_dropout_masks_nan_and_infinity(cuda):
    """Dropped and gated places are 0 whatever they hold; a NaN gate does not pass."""
    import torch
    import sushiblas_amd as sbx
    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 3.4e38, 1.0, -1.0, 0.0, -0.0] * 40,
                     device=cuda).reshape(10, 32)
    g = torch.tensor([1.0, 0.0, -1.0, float("nan"), float("inf"), 5e-45, -0.0, -float("inf")] * 40,
                     device=cuda).reshape(40, 8).roll(3, 0).reshape(10, 32).contiguous()
    for gate in (None, g):
        y = torch.empty_like(x)
        sbx.dropout(sbx.F32, 10, 32, x, 32, y, 32, 0.5, SEED, 5, gate=gate, ldg=32)
        want = ref.dropped(x.cpu().numpy(), 0.5, SEED, 5, None if gate is None else g.cpu().numpy())
        np.testing.assert_array_equal(y.cpu().numpy(), want)


def test_relu_forward_is_the_gate_on_itself(cuda):
    import torch
    import sushiblas_amd as sbx
    x = torch.randn((33, 77), device=cuda)
    y = x.clone()
    sbx.dropout(sbx.F32, 33, 77, y, 77, y, 77, 0.0, 0, 0, gate=y, ldg=77)
    assert torch.equal(y, x.clamp_min(0))


@pytest.mark.parametrize("gate", [False, True])
def test_dropout_gradient(cuda, gate):
    """The backward call's gradient against the formula and central differences
    of L = sum(w * dropout(relu?(x))) in fp64: L is linear away from 0, so the
    differences are off by rounding only -- L's few hundred terms of magnitude 1
    to 2^-52 over a step of 2^-10, below 1e-9."""
    import torch
    import sushiblas_amd as sbx
    rows, cols, p, h = 9, 21, 0.4, 2.0 ** -10
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((rows, cols), generator=gen, dtype=torch.float64)
    x = torch.where(x.abs() < 0.01, 0.5, x)
    w = torch.randn((rows, cols), generator=gen, dtype=torch.float64)

    def loss(x):
        d, y = x.to(cuda), torch.empty((rows, cols), dtype=torch.float64, device=cuda)
        sbx.dropout(sbx.F64, rows, cols, d, cols, y, cols, p, SEED, 8, gate=d if gate else None, ldg=cols)
        return float((y.cpu() * w).sum())

    dx = torch.empty((rows, cols), dtype=torch.float64, device=cuda)
    hx = x.clamp_min(0).to(cuda)
    sbx.dropout(sbx.F64, rows, cols, w.to(cuda), cols, dx, cols, p, SEED, 8,
                gate=hx if gate else None, ldg=cols)
    dx = dx.cpu()
    formula = w * torch.from_numpy(ref.keep(rows, cols, p, SEED, 8)) * (65536.0 / (65536 - ref.threshold(p)))
    if gate:
        formula = formula * (x > 0)
    assert torch.allclose(dx, formula, rtol=1e-15, atol=0)
    for i in range(0, rows * cols, 5):
        e = torch.zeros(rows * cols, dtype=torch.float64)
        e[i] = h
        e = e.reshape(rows, cols)
        assert abs((loss(x + e) - loss(x - e)) / (2 * h) - float(dx.reshape(-1)[i])) < 1e-9


def test_dropout_past_32_bit_offsets(cuda):
    """Rows whose byte offsets, and element offsets, pass 32 bits."""
    import torch
    import sushiblas_amd as sbx
    rows, cols, ld = 4, 100, (1 << 31) - 5
    x = torch.empty(3 * ld + cols, dtype=torch.bfloat16, device=cuda)
    host = torch.randn((rows, cols)).bfloat16()
    for r in range(rows):
        x[r * ld:r * ld + cols] = host[r].to(cuda)
    sbx.dropout(sbx.BF16, rows, cols, x, ld, x, ld, 0.2, SEED, 1)
    want = _rounded(ref.dropped(host.float().numpy(), 0.2, SEED, 1), torch.bfloat16)
    for r in range(rows):
        assert torch.equal(x[r * ld:r * ld + cols].cpu(), want[r])


def test_dropout_on_another_stream_and_in_a_graph(cuda):
    """A captured call replays to the eager result, with eager work between."""
    import torch
    import sushiblas_amd as sbx
    x = torch.randn((100, 333), device=cuda)
    want, y = torch.empty_like(x), torch.zeros_like(x)
    sbx.dropout(sbx.F32, 100, 333, x, 333, want, 333, 0.3, 77, 1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        sbx.dropout(sbx.F32, 100, 333, x, 333, y, 333, 0.3, 77, 1)
    s.synchronize()
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sbx.dropout(sbx.F32, 100, 333, x, 333, y, 333, 0.3, 77, 1)
    for i in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        sbx.dropout(sbx.F32, 100, 333, x, 333, want, 333, 0.3, 77, 1)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
