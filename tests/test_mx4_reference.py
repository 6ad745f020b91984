"""CPU checks of the plain implementations that the dropout and MXFP4 tests
compare against."""
import numpy as np
import pytest

import mx4_reference as ref


@pytest.mark.parametrize("counter,key,want", [
    # the known answers published with the generator (Salmon et al., SC'11)
    ((0, 0, 0, 0), 0, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (1 << 64) - 1, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), 0x299f31d0a4093822,
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_philox_known_answers(counter, key, want):
    assert tuple(int(x) for x in ref.philox(counter, key)) == want


def test_keep_rate():
    """The share kept lies within 5 standard deviations of 1 - p."""
    for p in (0.1, 0.5):
        n = 512 * 1000
        k = ref.keep(512, 1000, p, 12345, 3).mean()
        assert abs(k - (1 - p)) < 5 * np.sqrt(p * (1 - p) / n)


def test_every_representable_value_is_kept():
    """Values on the grid of their block come back as they were."""
    v = np.concatenate([ref.GRID, -ref.GRID, ref.GRID, -ref.GRID])[None, :]
    for e in (-127, -126, -3, 0, 100):
        assert np.array_equal(ref.fake(v * 2.0 ** e), v * 2.0 ** e)


@pytest.mark.parametrize("x,want", [(0.25, 0.0), (0.75, 1.0), (1.25, 1.0), (1.75, 2.0), (2.5, 2.0),
                                    (3.5, 4.0), (5.0, 4.0), (5.0001, 6.0), (6.5, 6.0), (7.9, 6.0)])
def test_rounding(x, want):
    """Ties go to the even code, and what is over 6 becomes 6."""
    v = np.zeros((1, 32))
    v[0, 0], v[0, 1], v[0, 2] = 4.0, x, -x
    assert list(ref.fake(v)[0, 1:3]) == [want, -want]


def test_pack_round_trip():
    rng = np.random.default_rng(5)
    v = ref.fake(rng.standard_normal((7, 300)))
    P, S = ref.pack(*ref.quantize(v), ldp=176, lds=64, fill=0xFF)
    assert np.array_equal(ref.unpack(P, S, 7, 300), v)
