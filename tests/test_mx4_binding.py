"""CPU checks of the leading dimensions that the Python binding passes for the
dropout and MXFP4 operators: a dimension of one entry, whose stride torch sets as
it likes, gets the packed one, and every other goes as it was given.

The library's calls are recorded, not made."""
import pytest
import torch

import sushiblas_amd as sbx


class Recorder:
    """Stands in for the loaded library; keeps the arguments of its one call."""

    def __getattr__(self, name):
        def call(*args):
            self.__dict__["called"], self.__dict__["args"] = name, args
            return 0
        return call


@pytest.fixture
def calls(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(sbx, "lib", lambda: r)
    return r


def _codes(rows, cols):
    """Scale codes laid out as documented, by torch's contiguous() from a row's side."""
    groups = -(-cols // 256)
    return torch.zeros((rows, groups, 8), dtype=torch.uint8).permute(1, 0, 2).contiguous()


def _elems(rows, cols):
    """Packed elements; a single row's as the transpose of a column."""
    w = 16 * -(-cols // 32)
    return torch.zeros((w, 1), dtype=torch.uint8).t() if rows == 1 else torch.zeros((rows, w), dtype=torch.uint8)


def _matrix(rows, cols):
    return torch.zeros((cols, 1)).t() if rows == 1 else torch.zeros((rows, cols))


def _fits(rows, cols, ldp, lds):
    """include/sbx.h's rule for an MXFP4 matrix."""
    return ldp % 16 == 0 and ldp >= 16 * -(-cols // 32) and lds % 8 == 0 and lds >= 8 * rows


SIZES = [(5, 1), (40, 31), (40, 32), (33, 255), (300, 256), (1, 40), (1, 1), (1, 300), (7, 257), (300, 1000)]


def test_torch_gives_one_group_a_stride_of_its_own():
    assert _codes(40, 256).stride(0) == 8 and _codes(40, 257).stride(0) == 320


@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize(calls, rows, cols):
    x, P, S, PT, ST = (_matrix(rows, cols), _elems(rows, cols), _codes(rows, cols), _elems(cols, rows),
                       _codes(cols, rows))
    sbx.mx4_quantize(sbx.F32, rows, cols, x, x.stride(0), P, P.stride(0), S, S.stride(0), PT, PT.stride(0), ST,
                     ST.stride(0), gate=x, ldg=x.stride(0), stream=0)
    a = calls.args
    assert calls.called == "sbx_mx4_quantize" and a[5] == a[7] == cols
    assert _fits(rows, cols, a[12], a[14]) and _fits(cols, rows, a[16], a[18])


@pytest.mark.parametrize("rows,cols", SIZES)
def test_dequantize(calls, rows, cols):
    y, P, S = _matrix(rows, cols), _elems(rows, cols), _codes(rows, cols)
    sbx.mx4_dequantize(sbx.F32, rows, cols, P, P.stride(0), S, S.stride(0), y, y.stride(0), stream=0)
    a = calls.args
    assert calls.called == "sbx_mx4_dequantize" and _fits(rows, cols, a[5], a[7]) and a[9] == cols


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("m,n", [(1, 7), (7, 1), (1, 1), (30, 50)])
@pytest.mark.parametrize("k", [1, 32, 256, 257, 700])
def test_gemm(calls, layout, m, n, k):
    A, SA, B, SB = _elems(m, k), _codes(m, k), _elems(n, k), _codes(n, k)
    C = _matrix(*((n, m) if layout else (m, n)))
    sbx.mx4_gemm(sbx.F32, layout, m, n, k, 1.0, A, A.stride(0), SA, SA.stride(0), B, B.stride(0), SB, SB.stride(0),
                 0.0, C, C.stride(0), stream=0)
    a = calls.args
    assert calls.called == "sbx_mx4_gemm"
    assert _fits(m, k, a[8], a[10]) and _fits(n, k, a[12], a[14]) and a[17] == (m if layout else n)


def test_dropout(calls):
    x = _matrix(1, 40)
    assert x.stride(0) == 1
    sbx.dropout(sbx.F32, 1, 40, x, x.stride(0), x, x.stride(0), 0.1, 1, 2, gate=x, ldg=x.stride(0), stream=0)
    a = calls.args
    assert calls.called == "sbx_dropout" and a[5] == a[7] == a[9] == 40


def test_other_leading_dimensions_go_as_given(calls):
    sbx.dropout(sbx.F32, 2, 40, 64, 41, 64, 43, 0.1, 1, 2, gate=64, ldg=42, stream=0)
    assert calls.args[5:10:2] == (41, 42, 43)
    sbx.mx4_quantize(sbx.F32, 300, 400, 64, 401, 64, 224, 64, 2408, 64, 176, 64, 3208, gate=64, ldg=403, stream=0)
    a = calls.args
    assert (a[5], a[7], a[12], a[14], a[16], a[18]) == (401, 403, 224, 2408, 176, 3208)
    sbx.mx4_dequantize(sbx.F32, 300, 400, 64, 224, 64, 2408, 64, 401, stream=0)
    assert calls.args[5:10:2] == (224, 2408, 401)
    sbx.mx4_gemm(sbx.F32, 0, 20, 30, 300, 1.0, 64, 176, 64, 168, 64, 192, 64, 248, 0.0, 64, 31, stream=0)
    a = calls.args
    assert (a[8], a[10], a[12], a[14], a[17]) == (176, 168, 192, 248, 31)
