"""CPU checks of the dropout and MXFP4 operators' largest sizes: what no launch can
take is refused as unsupported before any HIP call."""
import sushiblas_amd as sbx

SIDE = 1 << 30
ROW = 16 * (SIDE // 32)  # bytes of a packed row


def test_quantize():
    assert sbx.lib().sbx_mx4_quantize(0, sbx.BF16, SIDE, SIDE, 64, SIDE, 0, 0, 0.0, 1, 2, 64, ROW, 64, 8 * SIDE,
                                      64, ROW, 64, 8 * SIDE) == 2


def test_dequantize():
    assert sbx.lib().sbx_mx4_dequantize(0, sbx.BF16, SIDE, SIDE, 64, ROW, 64, 8 * SIDE, 64, SIDE) == 2


def test_gemm():
    for layout in (0, 1):
        assert sbx.lib().sbx_mx4_gemm(0, sbx.BF16, layout, SIDE, SIDE, 32, 1.0, 64, 16, 64, 8 * SIDE, 64, 16, 64,
                                      8 * SIDE, 0.0, 64, SIDE, 0) == 2
