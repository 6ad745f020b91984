"""CPU checks of the refusals of the norm, the few-token layer and the mixture of experts:
invalid arguments come back as a status before any HIP call."""
import pytest
import torch

import sushiblas_amd as sbx

BAD = -1 & (2**64 - 1)


def _norm(stream=0, dtype=0, rows=4, cols=40, X=64, ldx=40, R=64, ldr=40, W=64, eps=1e-6, H=64, ldh=40, Y=64,
          ldy=40, P=64, ldp=64, S=64, lds=32):
    return sbx.lib().sbx_rms_norm(stream, dtype, rows, cols, X, ldx, R, ldr, W, eps, H, ldh, Y, ldy, P, ldp, S, lds)


def _grad(stream=0, dtype=0, rows=4, cols=40, H=64, ldh=40, W=64, eps=1e-6, DY=64, lddy=40, DR=64, lddr=40, DX=64,
          lddx=40, DW=64, ws=64, size=1 << 30):
    return sbx.lib().sbx_rms_norm_grad(stream, dtype, rows, cols, H, ldh, W, eps, DY, lddy, DR, lddr, DX, lddx, DW,
                                       ws, size)


def _dequantize(stream=0, dtype=0, rows=4, cols=40, P=64, ldp=64, S=64, lds=32, Y=64, ldy=40):
    return sbx.lib().sbx_mx8_dequantize(stream, dtype, rows, cols, P, ldp, S, lds, Y, ldy)


def _linear(stream=0, dtype=0, m=4, n=6, k=40, alpha=1.0, X=64, ldx=64, SX=0, ldsx=32, B=64, ldb=32, SB=64, ldsb=48,
            beta=0.0, Y=64, ldy=6, epilogue=0):
    return sbx.lib().sbx_mx4_linear(stream, dtype, m, n, k, alpha, X, ldx, SX, ldsx, B, ldb, SB, ldsb, beta, Y, ldy,
                                    epilogue)


def _moe(stream=0, dtype=0, tokens=3, width=40, hidden=70, experts=5, topk=2, X=64, ldx=40, WR=64, ldwr=40,
         normalize=1, W1=64, ld1=32, S1=64, lds1=8 * 700, W2=64, ld2=48, S2=64, lds2=8 * 200, Y=64, ldy=40, chosen=64,
         weights=64, ws=64, size=1 << 30):
    return sbx.lib().sbx_mx4_moe(stream, dtype, tokens, width, hidden, experts, topk, X, ldx, WR, ldwr, normalize, W1,
                                 ld1, S1, lds1, W2, ld2, S2, lds2, Y, ldy, chosen, weights, ws, size)


ANY = [(dict(stream=BAD), 1), (dict(dtype=4), 2), (dict(dtype=-1), 2), (dict(dtype=1), 2)]
RECT = ANY + [(dict(rows=-1), 1), (dict(cols=-1), 1), (dict(rows=(1 << 30) + 1), 2), (dict(cols=(1 << 30) + 1), 2)]
EPS = [(dict(eps=-1e-9), 1), (dict(eps=float("nan")), 1), (dict(eps=float("inf")), 1)]
PACKED = [(dict(P=0), 1), (dict(P=72), 1), (dict(ldp=72), 1), (dict(ldp=32), 1), (dict(S=0), 1), (dict(S=68), 1),
          (dict(lds=24), 1), (dict(lds=36), 1)]


def dense(name, ld):
    return [({name: 0}, 1), ({name: 66}, 1), ({ld: 39}, 1)]


@pytest.mark.parametrize("kw,status", RECT + EPS + PACKED + dense("X", "ldx") + [
    (dict(R=66), 1), (dict(ldr=39), 1), (dict(W=0), 1), (dict(W=66), 1), (dict(H=66), 1), (dict(ldh=39), 1),
    (dict(Y=66), 1), (dict(ldy=39), 1), (dict(H=0, Y=0, P=0, S=0), 1), (dict(dtype=2, X=65), 1)])
def test_norm_refusals(kw, status):
    assert _norm(**kw) == status


@pytest.mark.parametrize("kw,status", RECT + EPS + dense("H", "ldh") + dense("DY", "lddy") + dense("DX", "lddx") + [
    (dict(W=0), 1), (dict(W=66), 1), (dict(DR=66), 1), (dict(lddr=39), 1), (dict(DW=66), 1), (dict(ws=0), 1),
    (dict(ws=72), 1), (dict(size=4 * 40 * 4 - 1), 1)])
def test_grad_refusals(kw, status):
    assert _grad(**kw) == status


@pytest.mark.parametrize("kw,status", RECT + PACKED + dense("Y", "ldy"))
def test_dequantize_refusals(kw, status):
    assert _dequantize(**kw) == status


@pytest.mark.parametrize("kw,status", ANY + [
    (dict(epilogue=2), 1), (dict(m=-1), 1), (dict(n=-1), 1), (dict(k=-1), 1), (dict(m=1025), 2),
    (dict(n=(1 << 30) + 1), 2), (dict(k=(1 << 23) + 1), 2), (dict(X=0), 1), (dict(X=66), 1), (dict(ldx=39), 1),
    (dict(SX=68), 1), (dict(SX=64, X=72), 1), (dict(SX=64, ldx=32), 1), (dict(SX=64, ldx=72), 1),
    (dict(SX=64, ldsx=24), 1), (dict(SX=64, ldsx=36), 1), (dict(B=0), 1), (dict(B=72), 1), (dict(ldb=16), 1),
    (dict(ldb=40), 1), (dict(SB=0), 1), (dict(SB=68), 1), (dict(ldsb=40), 1), (dict(Y=0), 1), (dict(Y=66), 1),
    (dict(ldy=5), 1), (dict(ldb=1 << 23), 2), (dict(SX=64, ldx=(1 << 26) + 16), 2),
    (dict(ldx=(1 << 24) + 1), 2), (dict(dtype=2, ldx=(1 << 25) + 1), 2), (dict(ldx=1 << 62), 2)])
def test_linear_refusals(kw, status):
    assert _linear(**kw) == status


@pytest.mark.parametrize("kw,status", ANY + [
    (dict(tokens=-1), 1), (dict(width=0), 1), (dict(hidden=0), 1), (dict(experts=0), 1), (dict(topk=0), 1),
    (dict(topk=6), 1), (dict(tokens=257), 2), (dict(width=(1 << 18) + 1), 2), (dict(hidden=(1 << 18) + 1), 2),
    (dict(experts=513), 2), (dict(experts=40, topk=17), 2),
    (dict(X=0), 1), (dict(X=66), 1), (dict(ldx=39), 1), (dict(WR=0), 1), (dict(WR=66), 1), (dict(ldwr=39), 1),
    (dict(W1=0), 1), (dict(W1=72), 1), (dict(ld1=16), 1), (dict(ld1=40), 1), (dict(S1=0), 1), (dict(S1=68), 1),
    (dict(lds1=8 * 699), 1), (dict(W2=0), 1), (dict(W2=72), 1), (dict(ld2=32), 1), (dict(S2=0), 1), (dict(S2=68), 1),
    (dict(lds2=8 * 199), 1), (dict(Y=0), 1), (dict(Y=66), 1), (dict(ldy=39), 1), (dict(chosen=66), 1),
    (dict(weights=66), 1), (dict(ws=0), 1), (dict(ws=72), 1), (dict(size=100), 1), (dict(ld1=1 << 23), 2),
    (dict(ld2=1 << 23), 2), (dict(ldx=1 << 21), 2), (dict(dtype=2, ldx=1 << 22), 2), (dict(ldx=1 << 62), 2)])
def test_moe_refusals(kw, status):
    assert _moe(**kw) == status


def test_noop_cases_need_no_device():
    assert _norm(rows=0) == 0 and _norm(cols=0) == 0 and _dequantize(rows=0) == 0 and _dequantize(cols=0) == 0
    assert _grad(rows=0, DW=0) == 0 and _grad(cols=0) == 0
    assert _linear(m=0) == 0 and _linear(n=0) == 0 and _moe(tokens=0) == 0


def test_workspaces():
    for rows in (1, 255, 256, 257, 10000):
        need = sbx.rms_norm_grad_workspace(rows, 40)
        assert 0 < need <= 4 * 40 * 256 and _grad(rows=rows, size=need - 1) == 1
    assert sbx.rms_norm_grad_workspace(0, 40) == 0 and sbx.rms_norm_grad_workspace(-1, 40) == 0
    need = sbx.mx4_moe_workspace(3, 40, 70, 5, 2)
    assert need > 0 and _moe(size=need - 1) == 1
    assert sbx.mx4_moe_workspace(3, 40, 70, 5, 6) == 0 and sbx.mx4_moe_workspace(257, 40, 70, 5, 2) == 0


def test_errors_raise_in_python():
    with pytest.raises(sbx.SbxError) as e:
        sbx.rms_norm(sbx.F32, 4, 4, 64, 4, 64, -1.0, Y=64, ldy=4, stream=0)
    assert e.value.status == 1
    ws = torch.zeros(5, dtype=torch.float32)  # too small, by its own size
    with pytest.raises(sbx.SbxError):
        sbx.rms_norm_grad(sbx.F32, 4, 40, 64, 40, 64, 1e-6, 64, 40, 64, 40, DW=64, workspace=ws, stream=0)


def test_shapes():
    assert sbx.mx8_shapes(5, 257) == ((5, 288), (2, 5, 8))


class Recorder:
    """Stands in for the loaded library; keeps the arguments of its one call."""

    def __getattr__(self, name):
        def call(*args):
            self.__dict__["called"], self.__dict__["args"] = name, args
            return 0
        return call


def test_leading_dimensions_of_single_entries(monkeypatch):
    """What torch gives a dimension of one entry goes as the packed one (two rows: as given)."""
    r = Recorder()
    monkeypatch.setattr(sbx, "lib", lambda: r)
    sbx.rms_norm(0, 1, 40, 64, 1, 64, 1e-6, R=64, ldr=1, H=64, ldh=1, Y=64, ldy=1, P=64, ldp=1, S=64, lds=8, stream=0)
    assert [r.args[i] for i in (5, 7, 11, 13, 15, 17)] == [40, 40, 40, 40, 64, 8]
    sbx.rms_norm(0, 2, 300, 64, 301, 64, 1e-6, P=64, ldp=400, S=64, lds=24, stream=0)
    assert [r.args[i] for i in (5, 15, 17)] == [301, 400, 24]
    sbx.rms_norm_grad(0, 1, 40, 64, 1, 64, 1e-6, 64, 1, 64, 1, DR=64, lddr=1, stream=0)
    assert [r.args[i] for i in (5, 9, 11, 13)] == [40] * 4
    sbx.mx8_dequantize(0, 1, 300, 64, 1, 64, 8, 64, 1, stream=0)
    assert [r.args[i] for i in (5, 7, 9)] == [320, 8, 300]
    sbx.mx4_linear(0, 1, 1, 40, 1.0, 64, 1, 64, 1, 64, 1, 0.0, 64, 1, stream=0)
    assert [r.args[i] for i in (7, 11, 13, 16)] == [40, 32, 8, 1]
    sbx.mx4_linear(0, 1, 9, 40, 1.0, 64, 1, 64, 48, 64, 8, 0.0, 64, 1, SX=64, ldsx=1, stream=0)
    assert [r.args[i] for i in (7, 9, 11, 13, 16)] == [64, 8, 48, 72, 9]
    sbx.mx4_moe(0, 1, 40, 70, 1, 1, 64, 1, 64, 1, 64, 32, 64, 8, 64, 48, 64, 8, 64, 1, stream=0)
    assert [r.args[i] for i in (8, 10, 13, 15, 17, 19, 21)] == [40, 40, 32, 8 * 140, 48, 8 * 40, 40]
