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


def refused(cache, step, *calls):
    """The calls of a step that no longer stands, refused before any operator is asked."""
    x = torch.zeros(step.rows, 1, 8)
    path = [[0][:n] for n in step.counts]
    run = dict(accept=lambda: cache.accept(step, path), append=lambda: cache.append(0, step, x, x),
               attention_into=lambda: cache.attention_into(0, step, x, x))
    before = books(cache)
    for name in calls:
        with pytest.raises(ValueError, match="latest" if name == "accept" else "stale"):
            run[name]()
    assert books(cache) == before


def stands(cache, step):
    """append and attention_into get as far as the operators, which refuse tensors on the CPU."""
    x = torch.zeros(step.rows, 1, 8)
    for call in (lambda: cache.append(0, step, x, x), lambda: cache.attention_into(0, step, x, x)):
        with pytest.raises(ValueError, match="current device"):
            call()


def test_steps_of_equal_lengths_are_told_apart():
    """A sequence that is back at the length which an earlier step left."""
    cache = make_cache()
    a, b = cache.add(), cache.add()
    cache.step([a], [10])
    old = cache.step([a], [4])
    cache.accept(old, [[0, 1]])
    new = cache.step([a], [2])
    assert cache.length(a) == 14
    refused(cache, old, "accept", "append", "attention_into")
    stands(cache, new)
    cache.trim(a, 10)  # its page goes to another sequence, and the length comes back
    cache.step([b], [5])
    later = cache.step([a], [4])
    assert cache.length(a) == 14
    refused(cache, old, "accept", "append", "attention_into")
    refused(cache, new, "accept", "append", "attention_into")
    cache.accept(later, [[0]])
    refused(cache, later, "accept", "append", "attention_into")


def test_steps_of_ended_sequences_are_refused():
    cache = make_cache()
    a, b = cache.add(), cache.add()
    both = cache.step([a, b], [4, 4])
    alone = cache.step([b], [2])
    cache.free(a)
    c = cache.add()
    cache.step([c], [4])  # a's page
    refused(cache, both, "accept", "append", "attention_into")
    stands(cache, alone)
    cache.accept(alone, [[0]])


def test_steps_whose_page_became_a_forks_are_refused():
    """The step's last page was shared with a fork, and its sequence got a copy when it went on."""
    cache = make_cache()
    cache._copy = lambda copies: None
    a = cache.add()
    step = cache.step([a], [6])
    f = cache.fork(a)
    stands(cache, step)
    more = cache.step([f], [1])  # (the fork's copy: a's pages are as they were)
    stands(cache, step)
    stands(cache, more)
    cache.fork(a)
    cache.step([a], [1])
    refused(cache, step, "accept", "append", "attention_into")


def test_steps_made_ahead_stand():
    """Chunks planned one after another are run in that order, and the last is accepted."""
    cache = make_cache()
    a, b = cache.add(), cache.add()
    steps = [cache.step([a, b], n) for n in ((5, 1), (3, 6), (2, 0))]
    for step in steps:
        stands(cache, step)
    for step in steps[:-1]:
        refused(cache, step, "accept")
    cache.accept(steps[-1], [[0, 1], []])
    assert (cache.length(a), cache.length(b)) == (10, 7)
    refused(cache, steps[-1], "accept")  # once


def test_steps_made_before_a_release_are_refused():
    """Pages that no later token sees may be ones that the step's own tokens see:
    the row before the next sees one row more."""
    cache = make_cache()
    a, b = cache.add(), cache.add()
    cache.step([a], [7])
    step = cache.step([a], [4])
    assert cache.release(a, 30) == 0
    stands(cache, step)  # (nothing was given up)
    assert cache.release(a, 4) == 2
    cache.step([b], [8])  # the pages that the window of the step's rows begins in
    refused(cache, step, "append", "attention_into")
    cache.accept(step, [[0, 1, 2, 3]])
    assert cache.length(a) == 11


def test_accept_copies_no_page_that_it_only_reads(monkeypatch):
    """After a fork the sequence gets pages of its own for its path's rows alone."""
    from nkilab import ops

    cache = make_cache(pages=4)
    copies, moves = [], []
    cache._copy = copies.extend
    monkeypatch.setattr(ops, "cache_accept", lambda k, v, table, lens, paths, **kw: moves.append((table.tolist(), paths.tolist())))
    a = cache.add()
    cache.step([a], [4])
    step = cache.step([a], [8])  # three pages of four
    f = cache.fork(a)
    cache.accept(step, [[0, 2]])
    assert copies == [(1, 3)] and moves == [([[0, 3, 2]], [[0, 2]])]
    assert cache.pages_of(a) == [0, 3] and cache.pages_of(f) == [0, 1, 2]
    assert (cache.length(a), cache.length(f), cache.free_pages()) == (6, 12, 0)
    # a path whose rows end where they begin needs no page at all
    step = cache.step([f], [0])
    cache.accept(step, [[]])
    assert (cache.length(f), cache.free_pages()) == (12, 0)


@pytest.mark.gpu
def test_accept_of_both_forks_reads_shared_pages():
    """Two sequences that share a step's pages keep paths of different lengths: a
    page that one only reads is not the one that the other writes."""
    from nkilab.cache import PagedCache

    import paged_reference as R

    cache = PagedCache(12, 1, 8, page_size=4, dtype=torch.float32)
    a = cache.add()
    rows = torch.randn(30, 1, 8, device="cuda")
    head = cache.step([a], [5])
    cache.append(0, head, rows[:5], rows[:5])
    f = cache.fork(a)
    both = cache.step([a, f], [12, 12])
    cache.append(0, both, rows[5:29], rows[5:29])
    g = cache.fork(f)
    cache.accept(both, [[1, 9], [0, 2, 5, 6, 8, 11]])
    at = lambda s: torch.stack([cache.k[0, p, :, o] for p, o in  # noqa: E731
                                (R.table_rows(cache.pages_of(s), 4, 12, j) for j in range(cache.length(s)))])
    assert torch.equal(at(a), rows[[0, 1, 2, 3, 4, 6, 14]])
    assert torch.equal(at(f), rows[[0, 1, 2, 3, 4] + [17 + i for i in (0, 2, 5, 6, 8, 11)]])
    assert torch.equal(at(g), torch.cat((rows[:5], rows[17:29])))


def test_accept_writes_lengths_apart_from_those_it_reads():
    """Every workgroup of a sequence reads its length, and one writes the new one:
    in the same place, the others might read that."""
    import ctypes

    from nkilab import _lib

    d = _lib.PagedCacheDesc(k=P, v=P, k_page=4096, k_head=1024, k_row=64, v_page=4096, v_head=1024, v_row=64, table=P,
                            table_row=8, lens=P + 400, q_start=None, pages=10, kv_heads=4, page_size=16, d=64, table_cols=8,
                            batch=3, rows=0, max_new=0, dtype=1)
    for new in (P + 400, P + 400 + 8, P + 400 - 8):
        assert _lib.lib().nkl_cache_accept(ctypes.byref(d), P, 4, 4, new, 1, 0, 0, None) == -1
        assert b"new_lens" in _lib.lib().nkl_last_error_string()


def test_books_need_no_assertions():
    """The same pages where Python runs without them."""
    import os
    import subprocess
    import sys

    import nkilab

    code = ("from nkilab.cache import PagePool; p = PagePool(8, 4); a = p.add(); p.own([a], [0], [9]); b = p.fork(a); "
            "print(p.own([a, b], [9, 9], [13, 10]), p.pages_of(a), p.pages_of(b), p.free_pages())")
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(nkilab.__file__)))
    out = [subprocess.run([sys.executable, *flags, "-c", code], env=env, capture_output=True, text=True, check=True).stdout
           for flags in ([], ["-O"])]
    assert out[0] == out[1] == "[(2, 3)] [0, 1, 3, 4] [0, 1, 2] 3\n"


def test_a_step_that_brings_a_sequence_nothing_leaves_its_draft_open():
    """Drafted nodes are accepted after a step of the batch in which their sequence had no rows."""
    cache = make_cache()
    a, b = cache.add(), cache.add()
    draft = cache.step([a], [5])
    other = cache.step([a, b], [0, 3])
    stands(cache, draft)
    cache.accept(other, [[], [0, 1]])
    stands(cache, draft)
    cache.accept(draft, [[0, 1]])
    assert (cache.length(a), cache.length(b)) == (2, 2)
    refused(cache, draft, "accept", "append", "attention_into")


def test_accept_moves_rows_where_they_are_now(monkeypatch):
    """A sequence that was given pages of its own since the step: its table of now counts."""
    from nkilab import ops

    cache = make_cache()
    cache._copy = lambda copies: None
    tables = []
    monkeypatch.setattr(ops, "cache_accept", lambda k, v, table, lens, paths, **kw: tables.append(table.tolist()))
    a = cache.add()
    step = cache.step([a], [6])
    f = cache.fork(a)
    assert cache.own([a], [0], [6], keep=True) == [(0, 2), (1, 3)]
    refused(cache, step, "append", "attention_into")
    cache.accept(step, [[1, 3]])
    assert tables == [[[2, 3]]] and cache.pages_of(f) == [0, 1]


def test_a_fork_of_no_sequence_adds_none():
    cache = make_cache()
    a = cache.add()
    before = books(cache)
    with pytest.raises(KeyError):
        cache.fork(a + 1)
    assert books(cache) == before and cache.add() == a + 1
