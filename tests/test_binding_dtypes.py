"""CPU checks that the Python binding's calls with fp32 and fp64 forms alone refuse
the other codes and tensors of other element sizes, instead of taking them for fp64
(whose kernels would read and write past a 16-bit tensor's end).

The library's calls are recorded, not made; a call that reaches it with such a
tensor's code has to be one that it refuses."""
import pytest
import torch

import sushiblas_amd as sbx


@pytest.fixture
def calls(monkeypatch):
    seen = []

    class Recorder:
        def __getattr__(self, name):
            return lambda *args: seen.append((name, args)) or 0

    monkeypatch.setattr(sbx, "lib", Recorder)
    return seen


@pytest.mark.parametrize("dtype", [sbx.BF16, sbx.F16, 4, -1])
def test_gemv_and_syrk_refuse_other_codes(calls, dtype):
    with pytest.raises(sbx.SbxError) as e:
        sbx.gemv(dtype, 0, 0, 2, 3, 1.0, 64, 3, 64, 1, 0.0, 64, 1, stream=0)
    assert e.value.status == 2
    with pytest.raises(sbx.SbxError) as e:
        sbx.syrk(dtype, 0, 0, 0, 3, 2, 1.0, 64, 2, 0, 0.0, 64, 3, 0, stream=0)
    assert e.value.status == 2
    assert not [n for n, _ in calls if n != "sbx_status_string"]


def test_gemv_and_syrk_take_their_own(calls):
    for dtype, gemv, syrk in ((sbx.F32, "sbx_sgemv", "sbx_ssyrk_strided_batched"),
                              (sbx.F64, "sbx_dgemv", "sbx_dsyrk_strided_batched")):
        sbx.gemv(dtype, 0, 0, 2, 3, 1.0, 64, 3, 64, 1, 0.0, 64, 1, stream=0)
        sbx.syrk(dtype, 0, 0, 0, 3, 2, 1.0, 64, 2, 0, 0.0, 64, 3, 0, stream=0)
        assert [n for n, _ in calls[-2:]] == [gemv, syrk]


@pytest.mark.parametrize("dt,code", [(torch.float32, sbx.F32), (torch.float64, sbx.F64), (torch.bfloat16, None),
                                     (torch.float16, None), (torch.uint8, None)])
def test_codes_of_tensors(calls, dt, code):
    t = torch.zeros(16, dtype=dt)
    sbx.relu(t, stream=0)
    sbx.fill_uniform(t, 1, 0, stream=0)
    sbx.fill_normal(t, 1, 0, stream=0)
    got = [args[1] for _, args in calls]
    assert len(got) == 3
    for g in got:
        assert g == code if code is not None else g not in (sbx.F32, sbx.F64)


def test_the_library_refuses_such_codes():
    assert sbx.lib().sbx_relu(0, -1, 64, 16) == 2
    assert sbx.lib().sbx_fill_uniform(0, -1, 64, 16, 1, 0) == 2
    assert sbx.lib().sbx_fill_normal(0, -1, 64, 16, 1, 0, 1.0) == 2
