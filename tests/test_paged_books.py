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


def make_cache(pages=16, page_size=4):
    """A cache on the CPU: its books work, and every operator refuses its tensors."""
    from nkilab.cache import PagedCache

    return PagedCache(pages, 1, 8, page_size=page_size, dtype=torch.float32, device="cpu")


def books(cache):
    return [list(t) for t in cache._tables.values()], list(cache._users), list(cache._free), dict(cache._lens), dict(cache._floor)


@pytest.mark.parametrize("call", ["compact", "step", "step of two", "accept", "tree"])
def test_a_refused_call_leaves_the_books_alone(call):
    """Where an operator refuses its part (here: tensors that are on no GPU) the
    sequences keep their pages and lengths, and the call can be made again."""
    cache = make_cache()
    a, b = cache.add(), cache.add()
    cache.step([a, b], [6, 6])
    if call == "compact":
        cache.free(a)
        run = cache.compact
    elif call == "step":
        c = cache.fork(a)
        run = lambda: cache.step([c], [1])  # noqa: E731
    elif call == "step of two":
        c = cache.fork(a)
        run = lambda: cache.step([b, c, a], [9, 1, 1])  # noqa: E731
    elif call == "accept":
        step = cache.step([a, b], [3, 4])
        cache.fork(b)
        run = lambda: cache.accept(step, [[0, 1], [0, 3]])  # noqa: E731
    else:
        run = lambda: cache.step([a], [3], tree=[[-1, 0, 0]])  # noqa: E731
    before = books(cache)
    for _ in range(2):
        with pytest.raises(ValueError, match="current device"):
            run()
        assert books(cache) == before
