"""Rotary scaling by turns over an original context so short that no pair turns often, with no GPU."""
import math

import pytest


@pytest.mark.parametrize("scaling", ["parts", "bands"])
@pytest.mark.parametrize("original", [1, 3, 6])
@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0)])
def test_every_pair_is_divided(scaling, original, dim, base):
    """The first pair turns original / (2 pi) times, below one: every frequency is divided by the factor."""
    from nkilab import ops

    plain = ops.Rotary(dim, base).frequencies
    r = ops.Rotary(dim, base, scaling=scaling, factor=8.0, original=original)
    assert r.frequencies == pytest.approx([f / 8 for f in plain], rel=1e-15)


@pytest.mark.parametrize("original", [7, 40, 201, 300])
def test_ends_of_the_ramp(original):
    """Kept: pairs that turn more often than high_turns; divided: less often than low_turns (to a
    whole pair's number, to which the ramp's ends are rounded outwards)."""
    from nkilab import ops

    plain = ops.Rotary(64).frequencies
    r = ops.Rotary(64, scaling="parts", factor=4.0, original=original)
    turns = [original * f / (2 * math.pi) for f in plain]
    step = plain[0] / plain[1]
    for t, f, p in zip(turns, r.frequencies, plain):
        assert p / 4 * (1 - 1e-15) <= f <= p
        if t > 32 * step:
            assert f == p
        if t < 1 / step:
            assert f == pytest.approx(p / 4, rel=1e-15)
