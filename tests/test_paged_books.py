"""The paged cache's books and refusals, with no GPU."""
import pytest
import torch

P = 1 << 20  # (an aligned address, refused before it is used)


def test_tree_mask_window_refusals():
    from nkilab import _lib, ops

    i32 = dict(dtype=torch.int32)
    parents, lens = torch.zeros(6, **i32), torch.zeros(2, **i32)
    for kw in (dict(window=0), dict(window=-1), dict(sinks=1), dict(window=3, sinks=-1), dict(window=3, sinks=1),
               dict(window=3, sinks=1, lens=lens[:1]), dict(window=3, sinks=1, lens=lens.long())):
        with pytest.raises(ValueError) as e:
            ops.tree_mask(parents, batch=2, **kw)
        assert "current device" not in str(e.value), kw
    with pytest.raises(ValueError, match="current device"):
        ops.tree_mask(parents, batch=2, window=3, sinks=1, lens=lens)
    mask = _lib.lib().nkl_tree_mask_window
    for window, sinks, lens in ((-1, 0, P), (0, 1, P), (3, -1, P), (3, 1, None)):
        assert mask(P, None, lens, 2, 6, 3, window, sinks, P, 1, None) == -1
    assert mask(None, None, None, 0, 0, 0, 3, 0, None, 1, None) == 0
