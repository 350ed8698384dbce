"""The operators of decoding in few bits together, as a user runs them: the decoder
block with 4-bit weights and rotary tables over an 8-bit cache, against the same
block in 64 bits over the rows that the cache then holds."""
import numpy as np
import pytest
import torch

import cache8_reference as R8
import paged_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# A block's outputs come of some ten roundings of its intermediate rows (half a step each), of
# relative size at most one beside the residual stream that they join: ten half steps, and 2^-13 for
# fp32 sums and softmax weights, of the largest output.
TOL = {t: 10 * torch.finfo(t).eps / 2 * (0 if t is torch.float32 else 1) + 2.0 ** -13 for t in DTYPES}


def make_block(seed=0, **kw):
    from nkilab.model import BlockConfig, DecoderBlock

    torch.manual_seed(seed)
    return DecoderBlock(BlockConfig(d_model=256, n_heads=4, n_kv_heads=2, d_ff=320, **kw)).eval()


def dense(block, weights):
    """The block's matrices in 64 bits, from 4-bit weights where there are any."""
    from nkilab import ops

    if weights is None:
        return {n: getattr(block, n).weight.detach().double().numpy() for n in ("wqkv", "wo", "wg", "wu", "wd")}
    gu = weights["gate_up"]
    side = lambda i: ops.W4Weight(gu.packed[i::2].contiguous(), gu.scales[i::2].contiguous(),  # noqa: E731
                                  None if gu.zeros is None else gu.zeros[i::2].contiguous(), gu.n, gu.k, gu.group)
    w = {"wqkv": weights["wqkv"], "wo": weights["wo"], "wg": side(0), "wu": side(1), "wd": weights["wd"]}
    return {n: ops.unpack_w4(t).double().cpu().numpy() for n, t in w.items()}


def norm(x, g, eps):
    return x / np.sqrt((x ** 2).mean(axis=1, keepdims=True) + eps) * g.detach().double().numpy()


def projected(block, w, x, pos):
    """(q, k, v) of rows x [T, 256] in 64 bits, q and k rotated."""
    cfg = block.cfg
    hd = cfg.head_dim
    qkv = norm(x, block.norm1.weight, cfg.eps) @ w["wqkv"].T
    q, k, v = np.split(qkv, [cfg.d_model, cfg.d_model + cfg.kv_heads * hd], axis=1)
    q, k, v = (t.reshape(len(x), -1, hd) for t in (q, k, v))
    if cfg.rotary is not None:
        q, k = R8.rotate(q, pos, cfg.rotary), R8.rotate(k, pos, cfg.rotary)
    return q, k, v


def rest(block, w, x, a):
    x1 = x + a.reshape(len(x), -1) @ w["wo"].T
    h = norm(x1, block.norm2.weight, block.cfg.eps)
    g = h @ w["wg"].T
    return x1 + (g / (1 + np.exp(-g)) * (h @ w["wu"].T)) @ w["wd"].T


def raw(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def step_and_check(block, weights, w, cache, step, x, starts, dtype, layer, bits=None, pos=None):
    """A decode step, held to the block over the rows that the cache holds after it."""
    from nkilab.model import nki_decode

    out = nki_decode(block, x.cuda(), cache, step, layer=layer, compute_dtype=dtype, weights=weights).double().cpu().numpy()
    xd = x.double().numpy()
    lens = step.lens.tolist()
    table = step.table.cpu().numpy()
    if pos is None:
        pos = np.concatenate([np.arange(n - (b - a), n) for n, a, b in zip(lens, starts, starts[1:])])
    q, k, v = projected(block, w, xd, pos)
    kc, ks, vc, vs = raw(cache.k[layer]), cache.k_scale[layer].cpu().numpy(), raw(cache.v[layer]), cache.v_scale[layer].cpu().numpy()
    kv, vv = R8.values(kc, ks), R8.values(vc, vs)
    # what was written: within half a code's step of the rows, which come with the block's own roundings
    for b, n in enumerate(lens):
        for i in range(starts[b + 1] - starts[b]):
            p, o = R.table_rows(table[b], cache.page_size, cache.pages, n - (starts[b + 1] - starts[b]) + i)
            for got, rows, s in ((kv, k, ks), (vv, v, vs)):
                row = rows[starts[b] + i]
                lim = np.abs(row) * 2.0 ** -4 + 2.0 ** -10 * 2.0 ** (s[p].astype(float) - 127)[:, None] + 2 * TOL[dtype] * np.abs(rows).max()
                assert (np.abs(got[p, :, o] - row) <= lim).all()
    a = R.attention(q, kv, vv, table, lens, starts, bits=bits, window=block.cfg.window, sinks=block.cfg.sinks)
    want = rest(block, w, xd, a)
    assert np.abs(out - want).max() <= TOL[dtype] * np.abs(want).max(), (np.abs(out - want).max(), np.abs(want).max())
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits4", [False, True])
def test_prompts_tokens_trees(dtype, bits4):
    """Prompts in chunks, single tokens, a drafted tree and its accepted path, a fork that both sides write to."""
    from nkilab import ops
    from nkilab.cache import PagedCache
    from nkilab.model import quantize_block

    rot = ops.Rotary(32, interleaved=True, scaling="bands", factor=4.0, original=64)
    block = make_block(rotary=rot)
    weights = quantize_block(block, group=64, zeros=True) if bits4 else None
    w = dense(block, weights)
    cache = PagedCache(40, 2, 64, layers=2, page_size=16, dtype=torch.float8_e4m3fn)
    a, b = cache.add(), cache.add()
    g = torch.Generator().manual_seed(1)
    rows = lambda n: torch.randn(n, 256, generator=g)  # noqa: E731
    run = lambda step, x, starts, **kw: step_and_check(block, weights, w, cache, step, x, starts, dtype, 1, **kw)  # noqa: E731
    run(cache.step([a, b], [37, 5]), rows(42), [0, 37, 42])
    run(cache.step([a, b], [1, 30]), rows(31), [0, 1, 31])
    for _ in range(3):
        run(cache.step([b, a], [1, 1]), 3 * rows(2), [0, 1, 2])
    tree = [[-1, 0, 0, 1, 3, 2, 4, 1], [-1, 0, 1]]
    ctx = [cache.length(a), cache.length(b)]
    depth = [[0, 1, 1, 2, 3, 2, 4, 2], [0, 1, 2]]
    step = cache.step([a, b], [8, 3], tree=tree)
    run(step, rows(11), [0, 8, 11], bits=[r for t in tree for r in R.tree_bits(t)],
        pos=np.concatenate([c + np.array(d) for c, d in zip(ctx, depth)]))
    before = R8.values(raw(cache.v[1]), cache.v_scale[1].cpu().numpy())
    path = [0, 1, 3, 4, 6]
    spots = [R.table_rows(cache.pages_of(a), 16, 40, ctx[0] + i) for i in path]
    cache.accept(step, [path, [0, 1, 2]])
    after = R8.values(raw(cache.v[1]), cache.v_scale[1].cpu().numpy())
    for i, (p, o) in enumerate(spots):
        q, u = R.table_rows(cache.pages_of(a), 16, 40, ctx[0] + i)
        x, y = before[p, :, o], after[q, :, u]
        # moved codes are the same but for those that became subnormal under a larger scale
        step_size = 2.0 ** -10 * 2.0 ** (cache.v_scale[1].cpu().numpy()[q].astype(float) - 127)[:, None]
        assert (np.abs(x - y) <= step_size).all()
    c = cache.fork(a)
    run(cache.step([a, c, b], [1, 4, 1]), rows(6), [0, 1, 5, 6])
    cache.free(b)
    cache.compact()
    run(cache.step([c, a], [1, 2]), 20 * rows(3), [0, 1, 3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_window_over_8_bits(dtype):
    from nkilab import ops
    from nkilab.cache import PagedCache

    block = make_block(rotary=ops.Rotary(64), window=20, sinks=3)
    w = dense(block, None)
    cache = PagedCache(20, 2, 64, page_size=8, dtype=torch.float8_e4m3fn)
    s = cache.add()
    x = torch.randn(60, 256, generator=torch.Generator().manual_seed(2))
    at = 0
    for n in (50, 1, 1, 7, 1):
        step_and_check(block, None, w, cache, cache.step([s], [n]), x[at:at + n], [0, n], dtype, 0)
        at += n
        cache.release(s, 20, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(dim=64), dict(dim=32, interleaved=True, scaling="parts", factor=8.0, original=32),
                                dict(dim=48, scaling="linear", factor=2.0)])
def test_forward_with_rotary_and_weights(dtype, kw):
    """nki_forward against the eager block, and nki_decode over a cache of the compute dtype against nki_forward."""
    from nkilab import ops
    from nkilab.cache import PagedCache
    from nkilab.model import nki_decode, nki_forward, quantize_block

    block = make_block(rotary=ops.Rotary(**kw))
    x = torch.randn(50, 256, generator=torch.Generator().manual_seed(3))
    want = block(x).detach()
    close = lambda out, ref: (out.cpu().double() - ref.double()).abs().max() <= TOL[dtype] * ref.abs().max()  # noqa: E731
    out = nki_forward(block, x.cuda(), compute_dtype=dtype)
    assert close(out, want)
    if dtype is torch.float32:
        assert close(nki_forward(block, x.cuda(), compute_dtype="split"), want)
    cache = PagedCache(10, 2, 64, page_size=16, dtype=dtype)
    s = cache.add()
    parts = [nki_decode(block, x[i:j].cuda(), cache, cache.step([s], [j - i]), compute_dtype=dtype) for i, j in ((0, 30), (30, 31), (31, 50))]
    assert close(torch.cat(parts), want)
    weights = quantize_block(block, group=32)
    w = dense(block, weights)
    with torch.no_grad():
        for n in ("wqkv", "wo", "wg", "wu", "wd"):
            getattr(block, n).weight.copy_(torch.from_numpy(w[n]))
    want = block(x).detach()
    assert close(nki_forward(block, x.cuda(), compute_dtype=dtype, weights=weights), want)


def test_refusals():
    from nkilab import ops
    from nkilab.cache import PagedCache
    from nkilab.model import BlockConfig, DecoderBlock, nki_decode, nki_forward, quantize_block

    with pytest.raises(ValueError):
        DecoderBlock(BlockConfig(d_model=64, n_heads=2, rotary=ops.Rotary(64)))
    with pytest.raises(ValueError):
        DecoderBlock(BlockConfig(d_model=64, n_heads=2, rotary=ops.Rotary(32), rope_base=100.0))
    block = make_block()
    weights = quantize_block(block)
    x = torch.randn(3, 256).cuda()
    with pytest.raises(ValueError, match="split"):
        nki_forward(block, x, compute_dtype="split", weights=weights)
    for bad in (dict(list(weights.items())[:3]), {**weights, "wo": weights["wd"]}, {**weights, "gate_up": weights["wo"]}):
        with pytest.raises(ValueError, match="4-bit"):
            nki_forward(block, x, weights=bad)
    cache = PagedCache(4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        nki_decode(block, x, cache, cache.step([cache.add()], [3]))


def test_captured_decode_step():
    """A step of one token a sequence captured, and replayed as the sequences grow within their pages."""
    from nkilab import ops
    from nkilab.cache import PagedCache
    from nkilab.model import nki_decode, quantize_block

    block = make_block(rotary=ops.Rotary(64))
    weights = quantize_block(block)
    caches = [PagedCache(8, 2, 64, page_size=64, dtype=torch.float8_e4m3fn) for _ in range(2)]
    prompt = torch.randn(30, 256, generator=torch.Generator().manual_seed(5)).cuda()
    for c in caches:
        s = [c.add(), c.add()]
        nki_decode(block, prompt, c, c.step(s, [20, 10]), compute_dtype="float16", weights=weights)
    x = torch.randn(2, 256).cuda()
    c = caches[0]
    step = c.step([0, 1], [1, 1])
    nki_decode(block, x, c, step, compute_dtype="float16", weights=weights)  # (and the workspaces are there)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nki_decode(block, x, c, step, compute_dtype="float16", weights=weights)
    for k in range(3):
        x.copy_(torch.randn(2, 256, generator=torch.Generator().manual_seed(k)))
        step.lens.copy_(torch.tensor([21 + k, 11 + k], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = nki_decode(block, x.clone(), caches[1], caches[1].step([0, 1], [1, 1]), compute_dtype="float16", weights=weights)
        assert torch.equal(out, want)
