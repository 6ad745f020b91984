"""GPU tests of sbx_mx4_gemm without terms (k = 0, or alpha = 0) on results of many
tiles: C = epilogue(beta * C), exact in every type, the operands not looked at; as
fast as a pass over C by tiles, not by single values."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("m,n", [(70, 90), (513, 700), (1500, 2051), (4096, 4100)])
def test_no_terms(cuda, name, layout, m, n):
    import torch
    import sushiblas_amd as sbx
    dt, code = {"f32": (torch.float32, sbx.F32), "bf16": (torch.bfloat16, sbx.BF16),
                "f16": (torch.float16, sbx.F16)}[name]
    rows, cols = (n, m) if layout else (m, n)
    c0 = torch.randint(-64, 64, (rows, cols + 3), generator=torch.Generator().manual_seed(m)).to(dt)
    for k, alpha, beta, relu in ((0, 1.0, 0.5, True), (300, 0.0, -0.5, False), (0, 2.0, 0.0, False)):
        c = c0.clone()
        if beta == 0:
            c[:, :cols] = float("nan")
        c = c.to(cuda)
        print("mx4_gemm", name, layout, m, n, k, alpha, beta, flush=True)
        sbx.mx4_gemm(code, layout, m, n, k, alpha, None, 0, None, 0, None, 0, None, 0, beta, c, cols + 3,
                     epilogue=sbx.EPILOGUE_RELU if relu else sbx.EPILOGUE_NONE)
        want = c0.clone()
        want[:, :cols] = (c0[:, :cols].float() * beta).to(dt)
        if relu:
            want[:, :cols].clamp_(min=0)
        assert torch.equal(c.cpu(), want)


def test_no_terms_costs_a_pass_over_the_result(cuda):
    """8192^2 in bf16, 268 MB to and fro, against torch's own pass over the same memory: within 3 times
    of it (single values of 16 x 16 blocks took 287 us, the tiles 55)."""
    import torch
    import sushiblas_amd as sbx
    n = 8192
    c = torch.zeros((n, n), dtype=torch.bfloat16, device=cuda)

    def best(f):
        times = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            f()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    own = best(lambda: sbx.mx4_gemm(sbx.BF16, 0, n, n, 0, 1.0, None, 0, None, 0, None, 0, None, 0, 0.5, c, n))
    theirs = best(lambda: c.mul_(0.5))
    print("us", own * 1e3, theirs * 1e3, flush=True)
    assert own < 3 * theirs
