"""GPU tests of the mixture's forms, as layer_sizes.py lists them (and test_layer_plan.py checks):
several groups of terms where waves have rows of their own, and choices among more experts than a wave
has lanes."""
import numpy as np
import pytest

import layer_reference as ref
import layer_sizes as sizes
from test_mx4_moe_gpu import Mixture, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("tokens,width,hidden,experts,topk", sizes.ROWS)
def test_mixtures_of_several_groups(cuda, name, tokens, width, hidden, experts, topk):
    Mixture(cuda, name, width, hidden, experts).check(_x(tokens, width), topk)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("tokens,experts,topk", sizes.CHOICES)
def test_choices(cuda, name, normalize, tokens, experts, topk):
    Mixture(cuda, name, 80, 48, experts).check(_x(tokens, 80), topk, normalize)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("experts", [68, 128, 131, 300])
@pytest.mark.parametrize("tokens", [1, 5, 9])
def test_equal_logits_of_far_experts_go_by_index(cuda, name, experts, tokens):
    """Equal ones among a lane's own and other lanes', as the highest of all; and all equal."""
    same = [e for e in (3, 67, 130, 195, 299) if e < experts] + [9, 40]
    m = Mixture(cuda, name, 96, 32, experts, same=same)
    x = 3.0 * m.wr[same[0]] * (1 + np.arange(tokens))[:, None]  # whose logits are the highest for experts like it
    order = ref.route(ref.rounded_to(x, m.dt), m.wr, len(same), True)[0]
    assert (order == np.sort(same)).all()
    m.check(x, len(same))
    m.check(x, 2, False)
    m.check(np.zeros((tokens, 96)), 12)


@pytest.mark.parametrize("ldx", [1 << 21, 1 << 40, 1 << 62])
def test_one_token_has_no_next_row(cuda, ldx):
    """Its leading dimension is not used: any is taken (of several tokens 2^23 bytes are refused)."""
    import torch
    import sushiblas_amd as sbx
    m = Mixture(cuda, "f32", 40, 30, 5)
    X = torch.randn(1, 40, device=cuda)
    Y, want = torch.zeros_like(X), torch.zeros_like(X)
    m.call(X, want, 2, True)
    size = sbx.mx4_moe_workspace(1, 40, 30, 5, 2)
    ws = torch.empty(size, dtype=torch.uint8, device=cuda)
    p = lambda t: t.data_ptr()  # noqa: E731
    args = (40, 30, 5, 2, p(X), ldx, p(m.WR), m.WR.shape[1], 1, p(m.W1), m.W1.shape[1], p(m.S1), m.S1.shape[1], p(m.W2),
            m.W2.shape[1], p(m.S2), m.S2.shape[1], p(Y), 40, None, None, p(ws), size)
    stream = torch.cuda.current_stream().cuda_stream
    assert sbx.lib().sbx_mx4_moe(stream, sbx.F32, 2, *args) != 0
    assert sbx.lib().sbx_mx4_moe(stream, sbx.F32, 1, *args) == 0
    torch.cuda.synchronize()
    assert torch.equal(Y, want)


@pytest.mark.parametrize("name", ref.TYPES)
@pytest.mark.parametrize("tokens,width,hidden,experts,topk", [(6, 300, 520, 9, 3), (40, 1024, 512, 16, 4), (30, 520, 96, 70, 2),
                                                              (150, 130, 300, 6, 2)])
def test_a_token_has_the_same_bits_anywhere(cuda, name, tokens, width, hidden, experts, topk):
    """In another place, among other tokens, of a call of the same sizes."""
    import torch
    m = Mixture(cuda, name, width, hidden, experts)
    X = ref.padded(cuda, _x(tokens, width), m.dt, 0)
    Y, got = torch.zeros_like(X), torch.zeros_like(X)
    m.call(X, Y, topk, True)
    order = torch.randperm(tokens, device=cuda, generator=torch.Generator(cuda).manual_seed(1))
    m.call(X[order].contiguous(), got, topk, True)
    assert torch.equal(got, Y[order])
    m.call(X[order.argsort()[:1]].repeat(tokens, 1), got, topk, True)
    assert all(torch.equal(got[i], got[0]) for i in range(tokens))
    others = ref.padded(cuda, _x(tokens, width, 3), m.dt, 0)
    others[tokens // 2] = X[1]
    m.call(others, got, topk, True)
    assert torch.equal(got[tokens // 2], Y[1])
