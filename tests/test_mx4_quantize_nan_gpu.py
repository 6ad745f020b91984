"""GPU tests of sbx_mx4_quantize on NaN of every kind: either sign, quiet or signalling, any
payload, alone or beside infinities, make their blocks NaN in both forms."""
import pytest

from test_mx4_quantize_gpu import _normal, _run, _types

pytestmark = pytest.mark.gpu

BITS = {
    "f32": [0x7FC00000, 0xFFC00000, 0x7F800001, 0xFF800001, 0xFFFFFFFF, 0x7FFFFFFF, 0xFF800000, 0x7F800000],
    "bf16": [0x7FC0, 0xFFC0, 0x7F81, 0xFF81, 0xFFFF, 0x7FFF, 0xFF80, 0x7F80],
    "f16": [0x7E00, 0xFE00, 0x7C01, 0xFC01, 0xFFFF, 0x7FFF, 0xFC00, 0x7C00],
}


@pytest.mark.parametrize("name", list(BITS))
def test_every_kind_of_nan(cuda, name):
    import torch
    dt, _ = _types(name)
    width = 32 if name == "f32" else 16
    ints = torch.int32 if name == "f32" else torch.int16
    bits = [b - (1 << width) if b >> (width - 1) else b for b in BITS[name]]
    x = _normal(150, 330, dt)
    raw = x.view(ints)
    for i, b in enumerate(bits):
        raw[3 + 17 * i, 5 + 37 * i] = b           # alone in its blocks
        raw[16 + 16 * i, 300] = bits[(i + 1) % 8]  # several in a column's
    raw[149, 320:330] = torch.tensor(bits + bits[:2], dtype=ints)
    _run(cuda, x, 330)
    _run(cuda, x, 330, p=0.3)
    g = _normal(150, 330, dt, 2)
    _run(cuda, x, 330, gate=g, p=0.1)
