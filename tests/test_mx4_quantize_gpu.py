"""GPU tests of sbx_mx4_quantize and sbx_mx4_dequantize against the plain
implementation (mx4_reference): codes are whole numbers, and what they stand for
is exact, so results have to be equal."""
import numpy as np
import pytest

import mx4_reference as ref

pytestmark = pytest.mark.gpu

SEED = 0xFEDCBA9876543210
TYPES = ["f32", "bf16", "f16"]


def _types(name):
    import torch
    import sushiblas_amd as sbx
    return {"f32": (torch.float32, sbx.F32), "bf16": (torch.bfloat16, sbx.BF16),
            "f16": (torch.float16, sbx.F16)}[name]


def _run(cuda, x, cols, gate=None, p=0.0, sid=3, pads=(0, 0, 0, 0), which="both", stream=None):
    """x, gate: host tensors (rows x at least cols); pads in units of 16 (P, PT)
    and 8 (S, ST) bytes.  Checks both forms and the bytes beside them."""
    import torch
    import sushiblas_amd as sbx
    code = {torch.float32: sbx.F32, torch.bfloat16: sbx.BF16, torch.float16: sbx.F16}[x.dtype]
    rows = x.shape[0]
    dx = x.to(cuda)
    dg = None if gate is None else gate.to(cuda)
    out = []
    for nr, nk, pp, ps, on in ((rows, cols, pads[0], pads[1], which != "cols"),
                               (cols, rows, pads[2], pads[3], which != "rows")):
        nb = (nk + 31) // 32
        ldp, lds = 16 * (nb + pp), 8 * (nr + ps)
        P = torch.full((nr, ldp), 0xA5, dtype=torch.uint8, device=cuda)
        S = torch.full(((nb + 7) // 8, lds), 0xA5, dtype=torch.uint8, device=cuda)
        out.append((P, ldp, S, lds) if on else (None, 0, None, 0))
    torch.cuda.synchronize()
    print("quantize", x.dtype, rows, cols, p, gate is not None, pads, which, flush=True)
    sbx.mx4_quantize(code, rows, cols, dx, x.shape[1], *out[0], *out[1], p=p, seed=SEED, stream_id=sid,
                     gate=dg, ldg=0 if gate is None else gate.shape[1], stream=stream)
    torch.cuda.synchronize()
    v = ref.dropped(x[:, :cols].float().numpy(), p, SEED, sid,
                    None if gate is None else gate[:, :cols].float().numpy())
    for (P, ldp, S, lds), w in zip(out, (v, v.T)):
        if P is not None:
            wp, ws = ref.pack(*ref.quantize(w), ldp=ldp, lds=lds, fill=0xA5)
            np.testing.assert_array_equal(P.cpu().numpy(), wp)
            np.testing.assert_array_equal(S.cpu().numpy(), ws)
    return out


def _normal(rows, cols, dt, seed=1):
    import torch
    gen = torch.Generator().manual_seed(seed)
    # magnitudes over many powers of two, some rows and columns large
    t = torch.randn((rows, cols), generator=gen) * torch.exp2(torch.randint(-6, 6, (rows, 1), generator=gen).float())
    return (t * torch.exp2(torch.randint(-3, 4, (1, cols), generator=gen).float())).to(dt)


SIZES = [(1, 1), (1, 33), (2, 64), (31, 31), (32, 256), (33, 257), (64, 8), (100, 300), (255, 129), (256, 64),
         (257, 511), (300, 1), (1, 1000), (520, 700), (1030, 520)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize_sizes(cuda, name, rows, cols):
    dt, _ = _types(name)
    x, g = _normal(rows, cols, dt), _normal(rows, cols, dt, 2)
    _run(cuda, x, cols)
    _run(cuda, x, cols, gate=g, p=0.3)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("which", ["rows", "cols"])
def test_quantize_one_form(cuda, name, which):
    dt, _ = _types(name)
    _run(cuda, _normal(130, 420, dt), 420, which=which)
    _run(cuda, _normal(130, 420, dt), 420, which=which, gate=_normal(130, 420, dt, 4), p=0.1)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("ldx,ldg,pads", [(301, 300, (1, 0, 0, 3)), (308, 303, (0, 5, 2, 0)), (300, 301, (3, 1, 1, 1))])
def test_quantize_leading_dimensions(cuda, name, ldx, ldg, pads):
    dt, _ = _types(name)
    _run(cuda, _normal(290, ldx, dt), 300, gate=_normal(290, ldg, dt, 3), p=0.2, pads=pads)


@pytest.mark.parametrize("p", [1e-7, 0.5, 1.0])
def test_quantize_rates(cuda, p):
    import torch
    _run(cuda, _normal(70, 260, torch.bfloat16), 260, p=p)
    _run(cuda, _normal(70, 260, torch.float32), 260, p=p)


def test_quantize_large(cuda):
    """Enough rows and columns for the forms that large matrices take."""
    import torch
    _run(cuda, _normal(2500, 2100, torch.bfloat16), 2100)
    _run(cuda, _normal(2049, 2307, torch.float32), 2307, gate=_normal(2049, 2307, torch.float32, 2), p=0.1)
    _run(cuda, _normal(2304, 2560, torch.float16), 2560, p=0.1)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_every_16_bit_value(cuda, name):
    """Every bf16 / f16 value (f32: their like and their neighbours) beside a
    largest one that makes each scale near it, ties and subnormals among them."""
    import torch
    dt, _ = _types(name)
    if name == "f32":
        bits = torch.arange(65536, dtype=torch.int64) << 16
        v = torch.cat([bits, bits | 1, (bits + 0xFFFF)]) & 0xFFFFFFFF
        v = torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32).view(torch.float32)
    else:
        v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt)
    v = v[torch.isfinite(v.float())]
    v = torch.cat([v, torch.zeros(-len(v) % 16, dtype=dt)]).reshape(-1, 16)
    # the block's other half: its largest, times 1 and 4, where that is finite
    top = v.float().abs().amax(1, keepdim=True)
    rows = []
    for f in (1.0, 4.0):
        t = (top * f).to(dt)
        t = torch.where(torch.isfinite(t.float()), t, top.to(dt))
        rows.append(torch.cat([v, t.expand(-1, 16)], 1))
    x = torch.cat(rows).contiguous()
    _run(cuda, x, 32)


def test_quantize_mixed_magnitudes_f32(cuda):
    """Random bit patterns of fp32, without infinities and NaN."""
    import torch
    gen = torch.Generator().manual_seed(11)
    x = torch.randint(-2 ** 31, 2 ** 31, (400, 512), generator=gen).to(torch.int32).view(torch.float32)
    x = torch.where(torch.isfinite(x), x, torch.zeros(()))
    _run(cuda, x, 512)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_infinity_and_nan(cuda, name):
    """A block with one of them is NaN, in each form its own; a masked one does not count."""
    import torch
    dt, code = _types(name)
    x = _normal(70, 100, dt)
    x[3, 40], x[50, 99], x[69, 0] = float("nan"), float("inf"), -float("inf")
    _run(cuda, x, 100)
    g = torch.ones((70, 100), dtype=dt)
    g[3, 40], g[69, 0] = 0.0, float("nan")
    out = _run(cuda, x, 100, gate=g)
    import sushiblas_amd as sbx
    y = torch.empty((70, 100), dtype=dt, device=cuda)
    sbx.mx4_dequantize(code, 70, 100, *out[0], y, 100)
    nan = torch.isnan(y.cpu())
    want = torch.zeros((70, 100), dtype=torch.bool)
    want[50, 96:] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("name", TYPES)
def test_quantize_zeros(cuda, name):
    """All-zero blocks, signs kept; and a matrix that dropout empties."""
    import torch
    dt, _ = _types(name)
    x = torch.zeros((40, 96), dtype=dt)
    x[:, 1::3] = -0.0
    x[7, 40] = 1.0
    _run(cuda, x, 96)
    _run(cuda, _normal(40, 96, dt), 96, p=1.0)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols,pads", [(1, 1, (0, 0, 0)), (3, 33, (1, 2, 1)), (40, 257, (0, 0, 3)),
                                            (129, 1000, (2, 1, 8)), (2000, 31, (0, 0, 0))])
def test_dequantize(cuda, name, rows, cols, pads):
    """Random codes, every scale among them."""
    import torch
    import sushiblas_amd as sbx
    dt, code = _types(name)
    rng = np.random.default_rng(rows + cols)
    nb = (cols + 31) // 32
    n = rng.integers(0, 16, (rows, nb, 32)).astype(np.uint8)
    sc = rng.integers(0, 256, (rows, nb)).astype(np.uint8)
    P, S = ref.pack(n, sc, ldp=16 * (nb + pads[0]), lds=8 * (rows + pads[1]), fill=0xFF)
    y = torch.full((rows, cols + pads[2]), 7.0, dtype=dt, device=cuda)
    sbx.mx4_dequantize(code, rows, cols, torch.from_numpy(P).to(cuda), P.shape[1],
                       torch.from_numpy(S).to(cuda), S.shape[1], y, cols + pads[2])
    with np.errstate(over="ignore"):
        want = torch.from_numpy(ref.values(n, sc, cols).astype(np.float32)).to(dt)
    got = y.cpu()
    assert torch.equal(torch.isnan(got[:, :cols]), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got[:, :cols], 1.0, 2.0, -2.0), torch.nan_to_num(want, 1.0, 2.0, -2.0))
    assert bool((got[:, cols:] == 7.0).all())


def test_quantize_past_32_bit_offsets(cuda):
    """Input rows, packed rows and code groups whose byte offsets pass 32 bits."""
    import torch
    import sushiblas_amd as sbx
    rows, cols, ld = 40, 70, 60_000_000  # 4.8e9 bytes of bf16
    x = torch.empty(rows * ld, dtype=torch.bfloat16, device=cuda)
    host = _normal(rows, cols, torch.bfloat16)
    for r in range(rows):
        x[r * ld:r * ld + cols] = host[r].to(cuda)
    ldp = 120_000_000  # 4.8e9 bytes
    P = torch.empty(rows * ldp, dtype=torch.uint8, device=cuda)
    S = torch.empty((1, rows, 8), dtype=torch.uint8, device=cuda)
    PT = torch.empty((cols, 32), dtype=torch.uint8, device=cuda)
    ST = torch.empty((1, cols, 8), dtype=torch.uint8, device=cuda)
    sbx.mx4_quantize(sbx.BF16, rows, cols, x, ld, P, ldp, S, 8 * rows, PT, 32, ST, 8 * cols)
    v = host.float().numpy()
    for w, p, s in ((v, torch.stack([P[r * ldp:r * ldp + 48] for r in range(rows)]), S), (v.T, PT, ST)):
        wp, ws = ref.pack(*ref.quantize(w))
        np.testing.assert_array_equal(p.cpu().numpy(), wp)
        np.testing.assert_array_equal(s.cpu().numpy().reshape(ws.shape), ws)
    y = torch.empty((rows, cols), device=cuda)
    sbx.mx4_dequantize(sbx.F32, rows, cols, P, ldp, S, 8 * rows, y, cols)
    np.testing.assert_array_equal(y.cpu().numpy(), ref.fake(v))
    # groups of codes 2^32 bytes apart
    cols = 600
    lds = (1 << 32) + 8
    S = torch.empty(2 * lds + 8 * rows, dtype=torch.uint8, device=cuda)
    host = _normal(rows, cols, torch.float32)
    P = torch.empty((rows, 304), dtype=torch.uint8, device=cuda)
    sbx.mx4_quantize(sbx.F32, rows, cols, host.to(cuda), cols, P, 304, S, lds)
    sbx.mx4_dequantize(sbx.F32, rows, cols, P, 304, S, lds, y := torch.empty((rows, cols), device=cuda), cols)
    np.testing.assert_array_equal(y.cpu().numpy(), ref.fake(host.numpy()))


def test_quantize_on_another_stream_and_in_a_graph(cuda):
    import torch
    import sushiblas_amd as sbx
    s = torch.cuda.Stream()
    _run(cuda, _normal(300, 400, torch.bfloat16), 400, p=0.1, stream=s)
    x = torch.randn((300, 400), device=cuda)
    bufs = [torch.empty(sh, dtype=torch.uint8, device=cuda)
            for sh in sbx.mx4_shapes(300, 400) + sbx.mx4_shapes(400, 300)]
    args = sum(((b, b.stride(0)) for b in bufs), ())
    sbx.mx4_quantize(sbx.F32, 300, 400, x, 400, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sbx.mx4_quantize(sbx.F32, 300, 400, x, 400, *args)
    for i in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = [b.clone() for b in bufs]
        sbx.mx4_quantize(sbx.F32, 300, 400, x, 400, *args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, bufs))
