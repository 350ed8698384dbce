"""Drafted trees under a window shorter than they are deep, on the GPU."""
import random

import pytest
import torch

from test_gpu_paged import DT, TOL, Batch, parents_of
from test_paged_cache import D, block_close, make_block, make_cache

pytestmark = pytest.mark.gpu


def branch(parents, i):
    return (branch(parents, parents[i]) if parents[i] >= 0 else []) + [i]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 2), (4, 14), (2, 11), (100, 3)])
@pytest.mark.parametrize("context", [(10, 30), (0, 1)])
def test_windowed_block_over_deep_trees(dtype, window, sinks, context):
    """Every node comes out as the windowed block's row over its own branch,
    however deep; a chain drafted as a tree as the same tokens in a chunk."""
    from nkilab.model import nki_decode

    block = make_block(window, sinks)
    cache = make_cache(dtype)
    rng = random.Random(7)
    parents = [list(range(-1, 5)), parents_of(rng, 20, "tree")]
    prompts = [torch.randn(n, D) for n in context]
    seqs = [cache.add(), cache.add()]
    run = lambda rows, step: nki_decode(block, rows.cuda(), cache, step, compute_dtype=dtype).cpu()  # noqa: E731
    run(torch.cat(prompts), cache.step(seqs, list(context)))
    plain = cache.fork(seqs[0])
    nodes = [torch.randn(len(p), D) for p in parents]
    out = run(torch.cat(nodes), cache.step(seqs, [6, 20], tree=parents)).split([6, 20])
    for prompt, par, x, o in zip(prompts, parents, nodes, out):
        for i in range(len(par)):
            whole = torch.cat([prompt] + [x[j:j + 1] for j in branch(par, i)])
            block_close(o[i], block(whole).detach()[-1], dtype)
    block_close(run(nodes[0], cache.step([plain], [6])), out[0], dtype)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (50, 4), (20, 45), (70, 200)])
def test_masks_under_a_window(dtype, window, sinks):
    """tree_mask with a window: of a node's ancestors those in its window and the
    sinks; the attention with these words is that of the node's branch."""
    from nkilab import ops

    lens, news = [20, 45, 300, 150, 3], [20, 16, 130, 64, 0]
    b = Batch(50, lens, news, 4, 2, 64, 16, dtype)
    rng = random.Random(51)
    parents = [parents_of(rng, n, kind) for n, kind in zip(news, ("chain", "star", "tree", "chain", "roots"))]
    flat = torch.tensor(sum(parents, []), dtype=torch.int32).cuda()
    at = dict(q_start=b.q_start, max_q=b.max_q)
    tree = ops.tree_mask(flat, **at, window=window, sinks=sinks, lens=b.lens)
    bits = []
    for length, n, par in zip(lens, news, parents):
        for i in range(n):
            path = branch(par, i)
            row = [0] * n
            for depth, j in enumerate(path):
                at_j = length - n + depth
                row[j] = int(at_j > length - n + len(path) - 1 - window or at_j < sinks)
            bits.append(row)
    for t, row in enumerate(bits):
        words = [sum(bit << i for i, bit in enumerate(row[64 * w:64 * w + 64])) for w in range(tree.shape[1])]
        assert [x % 2 ** 64 for x in tree[t].tolist()] == words, t
    out = ops.paged_attention(b.q, *b.args(), **at, tree=tree, window=window, sinks=sinks)
    b.check(out, window=window, sinks=sinks, bits=bits)
    chunk = ops.paged_attention(b.q, *b.args(), **at, window=window, sinks=sinks)
    for s, par in enumerate(parents):  # a chain is a prompt chunk, at any window
        if par == list(range(-1, news[s] - 1)) and par:
            rows = slice(b.starts[s], b.starts[s + 1])
            err = float((out[rows].float() - chunk[rows].float()).abs().max())
            assert err <= 2 * TOL[dtype] * float(b.vc.float().abs().max())


def test_captured_step_of_a_deep_tree():
    """A layer's calls for a tree deeper than the window, captured once and
    replayed over other rows, with eager calls between."""
    from nkilab.cache import PagedCache

    cache = PagedCache(40, 2, 64, layers=2, page_size=16, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(61)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()  # noqa: E731
    cache.k.zero_()
    cache.v.zero_()
    a, b = cache.add(), cache.add()
    cache.step([a, b], [30, 5])
    step = cache.step([a, b], [12, 7], tree=[list(range(-1, 11)), [-1, 0, 0, 1, 3, 4, 5]])
    k, v, q = r(19, 2, 64), r(19, 2, 64), r(19, 4, 64)
    o = torch.empty_like(q)

    def layer(i):
        turned = torch.empty_like(q)
        cache.append(i, step, k, v, q, turned, 10000.0)
        cache.attention_into(i, step, turned, o, window=4, sinks=8)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer(0)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        layer(0)
    for _ in range(4):
        for t in (k, v, q):
            t.copy_(r(*t.shape))
        cache.k[0, :, :, 3], cache.v[0, :, :, 3] = r(40, 2, 64), r(40, 2, 64)
        cache.k[1], cache.v[1] = cache.k[0], cache.v[0]
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        layer(1)
        assert torch.equal(got, o) and torch.equal(cache.k[0], cache.k[1])
