"""CPU checks of the dropout and MXFP4 entry points' refusals: invalid
arguments come back as a status before any HIP call."""
import pytest

import sushiblas_amd as sbx


def _dropout(stream=0, dtype=0, rows=4, cols=40, X=64, ldx=40, gate=0, ldg=0, Y=64, ldy=40, p=0.1,
             seed=1, sid=2):
    return sbx.lib().sbx_dropout(stream, dtype, rows, cols, X, ldx, gate, ldg, Y, ldy, p, seed, sid)


def _quantize(stream=0, dtype=0, rows=4, cols=40, X=64, ldx=40, gate=0, ldg=0, p=0.1, seed=1, sid=2,
              P=64, ldp=32, S=64, lds=32, PT=64, ldpt=16, ST=64, ldst=320):
    return sbx.lib().sbx_mx4_quantize(stream, dtype, rows, cols, X, ldx, gate, ldg, p, seed, sid, P, ldp,
                                      S, lds, PT, ldpt, ST, ldst)


def _dequantize(stream=0, dtype=0, rows=4, cols=40, P=64, ldp=32, S=64, lds=32, Y=64, ldy=40):
    return sbx.lib().sbx_mx4_dequantize(stream, dtype, rows, cols, P, ldp, S, lds, Y, ldy)


def _gemm(stream=0, dtype=0, layout=0, m=4, n=6, k=40, alpha=1.0, A=64, lda=32, SA=64, ldsa=32, B=64,
          ldb=32, SB=64, ldsb=48, beta=0.0, C=64, ldc=6, epilogue=0):
    return sbx.lib().sbx_mx4_gemm(stream, dtype, layout, m, n, k, alpha, A, lda, SA, ldsa, B, ldb, SB,
                                  ldsb, beta, C, ldc, epilogue)


ANY = [(dict(stream=-1 & (2**64 - 1)), 1), (dict(dtype=4), 2), (dict(dtype=-1), 2)]
RECT = ANY + [(dict(rows=-1), 1), (dict(cols=-1), 1), (dict(rows=(1 << 30) + 1), 2)]
DROP = RECT + [(dict(p=-0.1), 1), (dict(p=1.5), 1), (dict(p=float("nan")), 1), (dict(X=0), 1),
               (dict(X=66), 1), (dict(ldx=39), 1), (dict(gate=64, ldg=39), 1), (dict(gate=65, ldg=40), 1)]
PACKED = [(dict(P=0), 1), (dict(P=72), 1), (dict(ldp=24), 1), (dict(ldp=16), 1), (dict(S=0), 1),
          (dict(S=68), 1), (dict(lds=24), 1), (dict(lds=36), 1)]


@pytest.mark.parametrize("kw,status", DROP + [(dict(Y=0), 1), (dict(Y=65), 1), (dict(ldy=39), 1),
                                              (dict(dtype=1, X=68), 1)])
def test_dropout_refusals(kw, status):
    assert _dropout(**kw) == status


@pytest.mark.parametrize("kw,status", DROP + PACKED + [
    (dict(dtype=1), 2), (dict(P=0, S=0, PT=0, ST=0), 1), (dict(PT=0), 1), (dict(ST=0), 1), (dict(ldpt=8), 1),
    (dict(ldst=312), 1), (dict(PT=72), 1), (dict(ST=60), 1)])
def test_quantize_refusals(kw, status):
    assert _quantize(**kw) == status


@pytest.mark.parametrize("kw,status", RECT + PACKED + [(dict(dtype=1), 2), (dict(Y=0), 1), (dict(Y=66), 1),
                                                       (dict(ldy=39), 1)])
def test_dequantize_refusals(kw, status):
    assert _dequantize(**kw) == status


@pytest.mark.parametrize("kw,status", ANY + [
    (dict(dtype=1), 2), (dict(layout=2), 1), (dict(epilogue=2), 1), (dict(m=-1), 1), (dict(n=-1), 1),
    (dict(k=-1), 1), (dict(m=(1 << 30) + 1), 2), (dict(k=(1 << 23) + 1), 2), (dict(A=0), 1), (dict(A=72), 1),
    (dict(lda=16), 1), (dict(lda=40), 1), (dict(SA=0), 1), (dict(SA=68), 1), (dict(ldsa=24), 1),
    (dict(ldsa=36), 1), (dict(B=0), 1), (dict(B=72), 1), (dict(ldb=16), 1), (dict(SB=0), 1),
    (dict(ldsb=40), 1), (dict(C=0), 1), (dict(C=66), 1), (dict(ldc=5), 1), (dict(layout=1, ldc=3), 1),
    (dict(lda=1 << 23), 2), (dict(ldb=1 << 23), 2)])
def test_gemm_refusals(kw, status):
    assert _gemm(**kw) == status


def test_noop_cases_need_no_device():
    for f in (_dropout, _quantize, _dequantize):
        assert f(rows=0) == 0 and f(cols=0) == 0
    assert _gemm(m=0) == 0 and _gemm(n=0) == 0


def test_errors_raise_in_python():
    with pytest.raises(sbx.SbxError) as e:
        sbx.dropout(sbx.F32, 4, 4, 64, 4, 64, 4, 2.0, 1, 1, stream=0)
    assert e.value.status == 1


def test_shapes():
    assert sbx.mx4_shapes(5, 257) == ((5, 144), (2, 5, 8))
