"""Tables of rotary frequencies, and what the rotary entry points refuse, with no GPU."""
import math

import pytest
import torch


def test_frequencies():
    from nkilab import ops

    r = ops.Rotary(8, 100.0)
    assert r.frequencies == tuple(100.0 ** (-i / 4) for i in range(4)) and r.gain == 1.0
    assert ops.Rotary(8, 100.0, scaling="linear", factor=4.0).frequencies == tuple(f / 4 for f in r.frequencies)
    # the highest frequency stays, the lowest is divided by the factor
    b = ops.Rotary(8, 100.0, scaling="base", factor=4.0).frequencies
    assert b[0] == 1.0 and b[-1] == pytest.approx(r.frequencies[-1] / 4, rel=1e-14)
    assert ops.Rotary(2, 100.0, scaling="base", factor=4.0).frequencies == (1.0,)


@pytest.mark.parametrize("scaling", ["parts", "bands"])
def test_scaled_by_turns(scaling):
    """Pairs of many turns over the original context stay, those of few are divided, between is a monotone ramp."""
    from nkilab import ops

    plain = ops.Rotary(128, 10000.0).frequencies
    r = ops.Rotary(128, 10000.0, scaling=scaling, factor=8.0, original=4096)
    ratio = [f / p for f, p in zip(r.frequencies, plain)]
    high = 32 if scaling == "parts" else 4
    turns = [4096 * p / (2 * math.pi) for p in plain]
    assert ratio[0] == 1.0 and ratio[-1] == pytest.approx(1 / 8)
    assert all(a >= b for a, b in zip(ratio, ratio[1:]))
    for t, x in zip(turns, ratio):
        if t >= high * 1.5:
            assert x == 1.0
        if t <= 1 / 1.5:
            assert x == pytest.approx(1 / 8)
    assert r.gain == pytest.approx(0.1 * math.log(8) + 1 if scaling == "parts" else 1.0)
    assert ops.Rotary(128, scaling=scaling, factor=8.0, original=4096, magnitude=1.25).gain == 1.25


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=3), dict(dim=258), dict(dim=-2), dict(dim=64, base=1.0),
                                dict(dim=64, base=math.inf), dict(dim=64, base=math.nan), dict(dim=64, scaling="other"),
                                dict(dim=64, factor=2.0), dict(dim=64, scaling="linear", factor=0.5),
                                dict(dim=64, scaling="linear", factor=math.nan), dict(dim=64, scaling="parts", factor=2.0),
                                dict(dim=64, scaling="bands", factor=2.0, original=100, low_turns=4.0, high_turns=4.0),
                                dict(dim=64, scaling="bands", factor=2.0, original=100, low_turns=0.0),
                                dict(dim=64, magnitude=math.inf)])
def test_rotary_refuses(kw):
    from nkilab import ops

    with pytest.raises(ValueError):
        ops.Rotary(**kw)


def test_rotary_abi_refusals():
    from nkilab import _lib, ops

    L, P, good = _lib.lib(), 1 << 20, ops.Rotary(64)._packed

    def call(rotary=good, x=P, y=P + (1 << 16), H=2, S=3, d=64, st=(192, 64, 192, 64), positions=None, pos0=0, dtype=0):
        return L.nkl_rotary_apply(rotary, x, y, H, S, d, *st, positions, 0, pos0, 0, dtype, None)

    freq = [1.0] * _lib.ROTARY_PAIRS
    for bad in (dict(H=-1), dict(S=-1), dict(d=62), dict(st=(192, -64, 192, 64)), dict(rotary=None), dict(x=None),
                dict(y=None), dict(pos0=(1 << 31) - 2), dict(pos0=-(1 << 31) - 1), dict(y=P, st=(192, 64, 64, 128)),
                dict(rotary=_lib.pack_rotary(0, 0, 1.0, *freq)), dict(rotary=_lib.pack_rotary(129, 0, 1.0, *freq)),
                dict(rotary=_lib.pack_rotary(32, 0, math.nan, *freq)),
                dict(rotary=_lib.pack_rotary(32, 0, 1.0, *([1.5] + freq[1:]))),
                dict(rotary=_lib.pack_rotary(32, 0, 1.0, *([math.nan] + freq[1:])))):
        assert call(**bad) == -1, bad
    assert call(dtype=3) == -2
    assert call(H=0) == 0 and call(S=0, x=None, y=None) == 0


def test_rotary_into_refuses():
    from nkilab import ops

    r, x = ops.Rotary(64), torch.zeros(2, 3, 64)
    for y in (torch.zeros(2, 3, 65), torch.zeros(2, 3, 64, dtype=torch.bfloat16), torch.zeros(64, 3, 2).transpose(0, 2)):
        with pytest.raises(ValueError):
            ops.rotary_into(x, y, r)
    for pos in (torch.zeros(4, dtype=torch.int32), torch.zeros(3), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="positions"):
            ops.rotary_into(x, torch.zeros_like(x), r, positions=pos)
    with pytest.raises(ValueError, match="either"):
        ops.rotary_into(x, torch.zeros_like(x), r, positions=torch.zeros(3, dtype=torch.int32), pos0=1)
    with pytest.raises(ValueError, match="current device"):
        ops.rotary_into(x, torch.zeros_like(x), r)


def test_rotary_refuses_shared_rows():
    """An output whose rows lie in one place (an expanded tensor)."""
    from nkilab import _lib, ops

    L, P, r = _lib.lib(), 1 << 20, ops.Rotary(64)._packed
    for st in ((0, 64), (192, 0)):
        assert L.nkl_rotary_apply(r, P, P + (1 << 16), 2, 3, 64, 192, 64, *st, None, 0, 0, 0, 0, None) == -1
        assert b"share memory" in L.nkl_last_error_string()
