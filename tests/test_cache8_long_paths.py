"""Accepted paths that are too long for a cache of 8 bits are refused before anything happens, with no GPU."""
import pytest
import torch


def test_long_paths_are_refused_first():
    from nkilab import cache as C

    class Cache(C.PagedCache):
        def _copy(self, copies):
            assert not copies, "pages were copied"

    cache = Cache(pages=64, kv_heads=1, head_dim=16, page_size=64, dtype=torch.float8_e4m3fn, device="cpu")
    seq = cache.add()
    step = cache.step([seq], [1200])
    cache.fork(seq)  # (whose pages the path's rows may not be written to)
    books = lambda: ([list(t) for t in cache._tables.values()], list(cache._users), dict(cache._lens), list(cache._free))  # noqa: E731
    before = books()
    with pytest.raises(ValueError, match="1025 nodes"):
        cache.accept(step, [list(range(1, 1026))])
    assert books() == before
    cache.accept(step, [list(range(1100))])  # (in place: nothing moves)
    assert cache.length(seq) == 1100
