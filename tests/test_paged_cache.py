"""The page pool's books (on the host), and the decoder block over a paged cache (on the GPU)."""
import random

import numpy as np
import pytest
import torch

import paged_reference as R


def check_pool(pool):
    """Every page is free or in the tables that use it, and no two sequences own a row alone in one page."""
    users = [0] * pool.pages
    for table in pool._tables.values():
        assert len(set(p for p in table if p >= 0)) == sum(p >= 0 for p in table)
        for p in table:
            if p >= 0:
                users[p] += 1
    assert users == pool._users
    assert sorted(pool._free) == [p for p in range(pool.pages) if users[p] == 0]


@pytest.mark.parametrize("seed", range(20))
def test_pool_follows_a_model(seed):
    """Random adds, forks, appends, trims, releases and compactions, the rows'
    values kept beside them as plain lists."""
    from nkilab.cache import OutOfPages, PagePool

    rng = random.Random(seed)
    ps = rng.choice((1, 3, 8))
    pool = PagePool(60, ps)
    memory = [[None] * ps for _ in range(60)]
    rows = {}
    stamp = 0

    def copy(copies):
        old = [list(m) for m in memory]
        assert len({b for _, b in copies}) == len(copies) and not {b for _, b in copies} & {a for a, _ in copies}
        for a, b in copies:
            memory[b] = list(old[a])

    for _ in range(150):
        op = rng.choice(("add", "fork", "free", "append", "append", "append", "trim", "release", "compact"))
        seq = rng.choice(sorted(rows)) if rows else None
        if op == "add" or seq is None:
            rows[pool.add()] = []
        elif op == "fork":
            rows[pool.fork(seq)] = list(rows[seq])
        elif op == "free":
            pool.free(seq)
            del rows[seq]
        elif op == "append":
            seqs = rng.sample(sorted(rows), rng.randint(1, min(3, len(rows))))
            counts = [rng.randint(0, 7) for _ in seqs]
            before = ([list(t) for t in pool._tables.values()], list(pool._users), dict(pool._lens))
            try:
                copies = pool.own(seqs, [len(rows[s]) for s in seqs], [len(rows[s]) + n for s, n in zip(seqs, counts)])
            except OutOfPages:
                assert before == ([list(t) for t in pool._tables.values()], list(pool._users), dict(pool._lens))
                continue
            copy(copies)
            for s, n in zip(seqs, counts):
                for _ in range(n):
                    stamp += 1
                    page, off = R.table_rows(pool.pages_of(s), ps, pool.pages, len(rows[s]))
                    assert pool._users[page] == 1
                    memory[page][off] = stamp
                    rows[s].append(stamp)
        elif op == "trim":
            n = rng.randint(pool._floor[seq], len(rows[seq]))
            pool.trim(seq, n)
            rows[seq] = rows[seq][:n]
        elif op == "release":
            window, sinks = rng.randint(1, 20), rng.randint(0, 5)
            held = pool.pages_of(seq)
            pool.release(seq, window, sinks)
            for j in range(len(rows[seq])):
                if held[j // ps] >= 0 and R.table_rows(pool.pages_of(seq), ps, pool.pages, j) is None:
                    assert not any(R.sees(0, j, 1, n, window, sinks) for n in range(len(rows[seq]) + 1, len(rows[seq]) + 9))
        else:
            copy(pool.compact())
            used = pool.pages - pool.free_pages()
            assert all(p < used for t in pool._tables.values() for p in t)
        check_pool(pool)
        for s, values in rows.items():
            assert pool.length(s) == len(values)
            for j, value in enumerate(values):
                spot = R.table_rows(pool.pages_of(s), ps, pool.pages, j)
                assert spot is None or memory[spot[0]][spot[1]] == value
    assert stamp > 0


def test_pool_refusals():
    from nkilab.cache import OutOfPages, PagePool

    with pytest.raises(ValueError):
        PagePool(0, 16)
    with pytest.raises(ValueError):
        PagePool(4, 0)
    pool = PagePool(4, 4)
    a = pool.add()
    with pytest.raises(ValueError):
        pool.own([a, a], [0, 0], [1, 1])
    with pytest.raises(OutOfPages):
        pool.own([a], [0], [17])
    assert pool.free_pages() == 4 and pool.length(a) == 0
    pool.own([a], [0], [13])
    b = pool.fork(a)
    with pytest.raises(OutOfPages):  # the shared page that both write needs a copy
        pool.own([a, b], [13, 13], [14, 14])
    assert pool.release(a, 3) == 2 and pool.pages_of(a)[:2] == [-1, -1]
    with pytest.raises(ValueError):
        pool.trim(a, 12)
    with pytest.raises(ValueError):
        pool.own([a], [0], [1])
    with pytest.raises(ValueError):
        pool.release(a, 0)
    with pytest.raises(ValueError):
        pool.trim(b, 14)
    pool.free(b)
    assert pool.free_pages() == 2
    with pytest.raises(KeyError):
        pool.length(b)


# ----------------------------------------------------------------- on the GPU --

D, HEADS, KV, FF = 256, 4, 2, 512


def make_block(window=None, sinks=0, rope=10000.0, seed=0):
    from nkilab.model import BlockConfig, DecoderBlock

    torch.manual_seed(seed)
    return DecoderBlock(BlockConfig(d_model=D, n_heads=HEADS, d_ff=FF, n_kv_heads=KV, rope_base=rope, window=window,
                                    sinks=sinks)).eval()


def make_cache(dtype, pages=40, page_size=16, layers=2):
    from nkilab.cache import PagedCache

    return PagedCache(pages, KV, D // HEADS, layers, page_size, dtype)


# Relative to the largest value of the output.  fp32 runs differ in the order of
# fp32 sums of at most a thousand terms (2^-24 a step, under 2^-14 in all);
# 16-bit operands are rounded at each of the block's five products and at q, k,
# v and P, each by half a step of values near the output's own size: ten times
# eps / 2, doubled.
BLOCK_TOL = {torch.float32: 2.0 ** -14, torch.bfloat16: 10 * 2.0 ** -7, torch.float16: 10 * 2.0 ** -10}


def block_close(out, ref, dtype):
    ref = ref.double()
    err = float((out.double().cpu() - ref).abs().max())
    assert err <= BLOCK_TOL[dtype] * float(ref.abs().max()), (err, float(ref.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
@pytest.mark.parametrize("rope", [None, 10000.0])
def test_decode_gives_the_blocks_forward(dtype, window, sinks, rope):
    """Prompts of two sequences in chunks of uneven lengths, then single tokens,
    against the eager block over each whole sequence."""
    from nkilab.model import nki_decode, nki_forward

    block = make_block(window, sinks, rope)
    cache = make_cache(dtype)
    x = [torch.randn(n, D) for n in (70, 45)]
    want = [block(t).detach() for t in x]
    seqs = [cache.add(), cache.add()]
    done = [0, 0]
    got = [[], []]
    for counts in ((33, 1), (0, 30), (20, 3), (1, 1), (16, 10)):
        step = cache.step(seqs, counts)
        rows = torch.cat([t[a:a + n] for t, a, n in zip(x, done, counts)]).cuda()
        out = nki_decode(block, rows, cache, step, layer=1, compute_dtype=dtype)
        for i, part in enumerate(out.split(list(counts))):
            got[i].append(part.cpu())
        done = [a + n for a, n in zip(done, counts)]
    assert done == [70, 45] and [cache.length(s) for s in seqs] == done
    for g, w, t in zip(got, want, x):
        block_close(torch.cat(g), w, dtype)
        block_close(nki_forward(block, t.cuda(), compute_dtype=dtype), w, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
def test_drafted_tree_then_accepted_path(dtype, window, sinks):
    """A tree's nodes come out as the block's rows over their own branches; the
    accepted path's rows serve the tokens after it; a forked sequence and the
    compacted pool hold the same rows."""
    from nkilab.model import nki_decode

    block = make_block(window, sinks)
    cache = make_cache(dtype)
    prompts = [torch.randn(n, D) for n in (37, 16)]
    seqs = [cache.add(), cache.add()]
    run = lambda rows, step: nki_decode(block, rows.cuda(), cache, step, compute_dtype=dtype).cpu()  # noqa: E731
    run(torch.cat(prompts), cache.step(seqs, [37, 16]))
    spare = cache.fork(seqs[0])
    parents = [[-1, 0, 0, 1, 2, 2, 4], [-1, -1, 1, 2]]
    nodes = [torch.randn(len(p), D) for p in parents]
    step = cache.step(seqs, [7, 4], tree=parents)
    out = run(torch.cat(nodes), step).split([7, 4])

    def branch(parents, i):
        return (branch(parents, parents[i]) if parents[i] >= 0 else []) + [i]

    for prompt, par, x, o in zip(prompts, parents, nodes, out):
        for i in range(len(par)):
            whole = torch.cat([prompt] + [x[j:j + 1] for j in branch(par, i)])
            block_close(o[i], block(whole).detach()[-1], dtype)
    paths = [[0, 2, 4, 6], [1, 2]]
    cache.accept(step, paths)
    assert [cache.length(s) for s in seqs] == [41, 18]
    free = cache.free_pages()
    cache.compact()
    assert cache.free_pages() == free
    tail = torch.randn(3, D)  # one more token of each, and of the sequence forked before the tree
    out = run(tail, cache.step(seqs + [spare], [1, 1, 1]))
    kept = [torch.cat([p, x[path]]) for p, x, path in zip(prompts, nodes, paths)] + [prompts[0]]
    for i, rows in enumerate(kept):
        block_close(out[i], block(torch.cat([rows, tail[i:i + 1]])).detach()[-1], dtype)


@pytest.mark.gpu
def test_accept_after_a_fork_leaves_the_fork_alone():
    """A sequence forked while its nodes wait keeps them all."""
    cache = make_cache(torch.float32, layers=1)
    s = cache.add()
    step = cache.step([s], [20])
    k = torch.randn(20, KV, D // HEADS, device="cuda")
    cache.append(0, step, k, k)
    other = cache.fork(s)
    cache.accept(step, [[3, 7, 19]])
    rows = lambda q: torch.stack([cache.v[0, p, :, o] for p, o in  # noqa: E731
                                  (R.table_rows(cache.pages_of(q), 16, cache.pages, j) for j in range(cache.length(q)))])
    assert torch.equal(rows(s), k[[3, 7, 19]]) and torch.equal(rows(other), k)
    with pytest.raises(ValueError):
        cache.accept(step, [[3, 3]])
    with pytest.raises(ValueError):
        cache.accept(step, [[0], [1]])


@pytest.mark.gpu
def test_released_pages_serve_other_sequences():
    """Under a window, pages that no later token sees go to another sequence while the first goes on."""
    from nkilab.model import nki_decode

    block = make_block(window=20, sinks=3)
    cache = make_cache(torch.float32, pages=8, layers=1)
    x = torch.randn(100, D)
    a = cache.add()
    nki_decode(block, x[:90].cuda(), cache, cache.step([a], [90]))
    assert cache.free_pages() == 2 and cache.release(a, 20, 3) == 3
    b = cache.add()
    y = torch.randn(60, D)
    out = nki_decode(block, torch.cat((x[90:], y)).cuda(), cache, cache.step([a, b], [10, 60])).cpu()
    block_close(out[:10], block(x).detach()[90:], torch.float32)
    block_close(out[10:], block(y).detach(), torch.float32)


@pytest.mark.gpu
def test_decode_refusals():
    from nkilab.model import nki_decode

    block, cache = make_block(), make_cache(torch.bfloat16)
    s = cache.add()
    step = cache.step([s], [2])
    x = torch.randn(2, D).cuda()
    for kw in (dict(compute_dtype="split"), dict(), dict(compute_dtype="float16")):  # the cache is bf16
        with pytest.raises(ValueError):
            nki_decode(block, x, cache, step, **kw)
    with pytest.raises(ValueError):
        nki_decode(block, x[:1], cache, step, compute_dtype="bfloat16")
    for kw in (dict(counts=[1, 1]), dict(counts=[-1]), dict(counts=[2], tree=[[-1]])):
        with pytest.raises(ValueError):
            cache.step([s], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["flash", "naive"])
def test_windowed_block_forward(variant):
    from nkilab.model import nki_forward

    block = make_block(window=33, sinks=2)
    x = torch.randn(150, D)
    if variant == "naive":
        with pytest.raises(ValueError, match="window"):
            nki_forward(block, x.cuda(), attention_variant=variant)
    else:
        want = block(x).detach()
        block_close(nki_forward(block, x.cuda(), attention_variant=variant), want, torch.float32)
        block_close(nki_forward(block, x.cuda(), compute_dtype="split"), want, torch.float32)
        assert np.allclose(nki_forward(block, x.numpy()), want.numpy(), atol=1e-3)


def test_stale_steps_are_refused():
    """A step is of use until its cache is compacted, and accepted once, as the
    latest of its sequences."""
    from nkilab.cache import PagedCache

    cache = PagedCache(16, 1, 8, page_size=4, dtype=torch.float32, device="cpu")
    cache._copy = lambda copies: None
    a, b = cache.add(), cache.add()
    cache.step([a], [9])
    old = cache.step([b], [3])
    new = cache.step([b], [5])
    with pytest.raises(ValueError, match="latest"):
        cache.accept(old, [[0]])
    assert cache.length(b) == 8
    cache.accept(new, [[0, 1]])
    assert cache.length(b) == 5
    with pytest.raises(ValueError, match="latest"):
        cache.accept(new, [[0, 1]])
    step = cache.step([b], [2])
    assert cache.compact() == []  # nothing moved: the step stands
    cache.accept(step, [[0]])
    step = cache.step([b], [2])
    cache.free(a)
    assert cache.compact()
    x = torch.zeros(2, 1, 8)
    for call in (lambda: cache.accept(step, [[0]]), lambda: cache.append(0, step, x, x),
                 lambda: cache.attention_into(0, step, x, x)):
        with pytest.raises(ValueError, match="stale"):
            call()
    assert cache.length(b) == 8


def test_accept_after_a_release_changes_nothing():
    """A path that would leave a sequence shorter than when it gave up pages is
    refused before any sequence is changed."""
    from nkilab.cache import PagedCache

    cache = PagedCache(16, 1, 8, page_size=4, dtype=torch.float32, device="cpu")
    a, b = cache.add(), cache.add()
    step = cache.step([a, b], [12, 20])
    assert cache.release(b, 8) == 3
    books = [cache.pages_of(s) for s in (a, b)]
    with pytest.raises(ValueError, match="gave up pages"):
        cache.accept(step, [list(range(5)), list(range(7))])
    assert [cache.length(s) for s in (a, b)] == [12, 20] and [cache.pages_of(s) for s in (a, b)] == books
    cache.accept(step, [list(range(5)), list(range(20))])
    assert [cache.length(s) for s in (a, b)] == [5, 20]


@pytest.mark.parametrize("kind", [list, tuple, np.array, torch.tensor])
def test_accept_takes_any_sequence_of_nodes(kind):
    from nkilab.cache import PagedCache

    cache = PagedCache(4, 1, 8, page_size=4, dtype=torch.float32, device="cpu")
    a = cache.add()
    step = cache.step([a], [6])
    for bad in ([1, 0], [0, 6], [-1, 0], [2, 2]):
        with pytest.raises(ValueError, match="ascend"):
            cache.accept(step, [kind(bad)])
    cache.accept(step, [kind([0, 1, 2])])
    assert cache.length(a) == 3


@pytest.mark.parametrize("parents", [[0, 0], [-1, 1], [-2, 0], [-1, 0, 5]])
def test_trees_that_are_none_are_refused(parents):
    from nkilab.cache import PagedCache

    cache = PagedCache(4, 1, 8, page_size=4, dtype=torch.float32, device="cpu")
    a = cache.add()
    with pytest.raises(ValueError, match="parents"):
        cache.step([a], [len(parents)], tree=[parents])
    assert cache.length(a) == 0 and cache.free_pages() == 4
