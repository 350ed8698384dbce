"""Each route that the attention over a paged cache can take -- rows of a tile,
whole or split keys, pages that half tiles fit or do not -- with the masks,
values and layouts at which it can go wrong."""
import random

import numpy as np
import pytest
import torch

import paged_reference as R
from test_gpu_paged import DT, TOL, Batch, close, parents_of

gpu = pytest.mark.gpu

MANY = [(31 * i * i) % 560 + 40 for i in range(20)]

# name: lens, news, H, Hkv, and whether 16-bit calls split their keys.  Wide
# routes have more than 32 rows to a K/V head; "one" has more of their tiles
# than 256 CUs and keys too few to be split, "few" has fewer tiles, "split" keys
# enough, of several sequences or one (whose items fill ranges of their own).
ROUTES = {
    "wide_one": (MANY, [min(n, 33 + 7 * (i % 14)) for i, n in enumerate(MANY)], 16, 8, False),
    "wide_few": ([300, 61], [90, 61], 4, 2, False),
    "wide_split": ([2600, 900, 40], [70, 5, 40], 4, 2, True),
    "wide_split_alone": ([3000], [40], 4, 4, True),
    "narrow_one": (MANY, [1 + i % 5 for i in range(20)], 8, 8, False),
    "narrow_split": ([2600, 900, 40], [7, 1, 3], 4, 2, True),
    "narrow_split_alone": ([3000], [1], 6, 2, True),
}
WINDOWS = ((None, 0), (45, 20), (1400, 40))  # (the last leaves the long sequences' keys split)


def batch(route, dtype, d, page, seed=40, layout="page_major"):
    """The route's batch; checks that the call takes the route."""
    from nkilab import _lib

    lens, news, H, Hkv, split = ROUTES[route]
    b = Batch(seed, lens, news, H, Hkv, d, page, dtype, layout=layout)
    if dtype != "fp32":
        desc = _lib.pack_cache(b.kc.data_ptr(), b.vc.data_ptr(), *b.kc.stride()[:3], *b.vc.stride()[:3],
                               b.table.data_ptr(), b.table.stride(0), b.lens.data_ptr(), b.q_start.data_ptr(), *b.kc.shape,
                               b.table.shape[1], len(lens), b.starts[-1], b.max_q, {"bf16": 1, "fp16": 2}[dtype])
        for window, sinks in ((None, 0), (1400, 40)):
            need = _lib.lib().nkl_paged_attention_workspace_bytes(desc, H, window or 0, sinks, 0)
            assert (need > 0) == split
    if route == "wide_one":
        tiles = -(-b.max_q * (H // Hkv) // 128) * len(lens) * Hkv
        assert tiles > torch.cuda.get_device_properties(0).multi_processor_count
    return b


def attention(b, window=None, sinks=0, bits=None):
    """R.attention of the batch, whole sequences and heads at a time."""
    q, kc, vc = (t.double().cpu().numpy() for t in (b.q, b.kc, b.vc))
    out = np.full(q.shape, np.nan)
    group = b.H // b.Hkv
    for s, length in enumerate(b.lens_host):
        t0, n = b.starts[s], b.starts[s + 1] - b.starts[s]
        if n == 0:
            continue
        spots = [R.table_rows(b.table_host[s], b.page, b.pages, j) for j in range(length)]
        there = np.array([x is not None for x in spots], bool)
        P, O = np.array([x if x is not None else (0, 0) for x in spots], int).reshape(-1, 2).T
        j, ctx = np.arange(length), length - n
        pos = ctx + np.arange(n)
        if bits is None:
            seen = j[None] <= pos[:, None]
        else:
            m = np.array([row[:n] for row in bits[t0:t0 + n]], bool)
            pos = ctx - 1 + m.sum(1)
            seen = np.ones((n, length), bool)
            seen[:, max(ctx, 0):] = m[:, max(-ctx, 0):]
        if window:
            near = (j[None] > pos[:, None] - window) | (j[None] < sinks)
            seen &= near if bits is None else near | (j[None] >= ctx)
        seen &= there[None]
        k, v = kc[P, :, O].repeat(group, 1).transpose(1, 0, 2), vc[P, :, O].repeat(group, 1).transpose(1, 0, 2)
        with np.errstate(invalid="ignore", over="ignore"):
            sc = q[t0:t0 + n].transpose(1, 0, 2) @ k.transpose(0, 2, 1) / np.sqrt(b.d)
            sc = np.where(seen[None], sc, -np.inf)
            top = sc.max(-1, keepdims=True, initial=-np.inf)
            w = np.where(seen[None], np.exp(sc - np.where(np.isfinite(top), top, 0)), 0)
            odd = ~np.isfinite(v)
            o = w @ np.where(odd, 0, v)
            for x in (odd.any((0, 2)) & seen.any(0)).nonzero()[0]:  # (0 inf of a key that is not seen is no NaN)
                o[:, seen[:, x]] += np.where(odd[:, x], v[:, x], 0)[:, None]
            total = w.sum(-1, keepdims=True)
            o = np.where(seen.any(-1)[None, :, None], o / np.where(total > 0, total, 1), 0)
        out[t0:t0 + n] = o.transpose(1, 0, 2)
    return out


def check(b, out, **kw):
    close(out, attention(b, **kw), b.dtype, float(b.vc.float().abs().max()))


def test_the_reference_is_the_definition():
    """attention() against R.attention, on the CPU."""
    b = Batch.__new__(Batch)
    g = torch.Generator().manual_seed(44)
    b.kc, b.vc = torch.randn(9, 2, 4, 8, generator=g), torch.randn(9, 2, 4, 8, generator=g)
    b.table_host, b.lens_host, b.starts = [[3, 0, -1, 7], [8, 1, 2, 11], [4, 5, 6, -1]], [15, 16, 2], [0, 5, 12, 15]
    b.q = torch.randn(15, 4, 8, generator=g)
    b.page, b.pages, b.H, b.Hkv, b.d, b.dtype = 4, 9, 4, 2, 8, "fp32"
    rng = random.Random(45)
    tree = sum((R.tree_bits(parents_of(rng, n, "tree")) for n in (5, 7, 3)), [])
    b.vc[8, 0, 1, 3], b.vc[0, 1, 2] = np.inf, np.nan
    for bits in (None, tree):
        for kw in ({}, dict(window=3, sinks=2), dict(window=1), dict(window=9, sinks=6)):
            with np.errstate(invalid="ignore"):
                want = R.attention(b.q, b.kc, b.vc, b.table_host, b.lens_host, b.starts, bits=bits, **kw)
            got = attention(b, bits=bits, **kw)
            assert np.array_equal(np.isfinite(got), np.isfinite(want))
            assert np.allclose(got, want, rtol=1e-12, atol=1e-12, equal_nan=True)


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("d,page", [(24, 16), (24, 100), (64, 32), (64, 24), (128, 64), (128, 40)])
@pytest.mark.parametrize("route", list(ROUTES))
def test_routes(route, d, page, dtype):
    from nkilab import ops

    b = batch(route, dtype, d, page, layout="row_major" if d == 64 else "page_major")
    for window, sinks in WINDOWS:
        kw = dict(q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
        out = ops.paged_attention(b.q, *b.args(), **kw)
        check(b, out, window=window, sinks=sinks)
        # rows as columns of a wider tensor, an output of uneven rows, the same bits every time
        wide = torch.cat((torch.full_like(b.q, 9.0), b.q), dim=2)
        o = torch.full((b.H, b.q.shape[0], d + 8), 7.0, dtype=DT[dtype], device="cuda")
        ops.paged_attention_into(wide[:, :, d:], o[:, :, :d].transpose(0, 1), *b.args(), **kw)
        assert torch.equal(o[:, :, :d].transpose(0, 1), out) and (o[:, :, d:] == 7).all()


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("page", [32, 40])
@pytest.mark.parametrize("route", list(ROUTES))
def test_routes_under_trees(route, page, dtype):
    from nkilab import ops

    b = batch(route, dtype, 64, page)
    rng = random.Random(41)
    news = ROUTES[route][1]
    parents = [parents_of(rng, n, ("tree", "chain", "roots", "star")[i % 4]) for i, n in enumerate(news)]
    tree = ops.tree_mask(torch.tensor(sum(parents, []), dtype=torch.int32).cuda(), q_start=b.q_start, max_q=b.max_q)
    bits = sum((R.tree_bits(p) for p in parents), [])
    for window, sinks in WINDOWS:
        out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, tree=tree, window=window, sinks=sinks)
        check(b, out, window=window, sinks=sinks, bits=bits)


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("page", [32, 40])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), "lowest"])
@pytest.mark.parametrize("route", list(ROUTES))
def test_routes_with_masked_values(route, value, page, dtype):
    """Keys that no row of a sequence sees, rows behind its last, and one that
    only its last row sees (V) hold a value that is none, or the type's lowest:
    the other rows do not know of it."""
    from nkilab import ops

    b = batch(route, dtype, 64, page, seed=42)
    lens, news, _, _, split = ROUTES[route]
    window, sinks = (1400, 2) if split else (30, 2)
    if value == "lowest":
        value = torch.finfo(DT[dtype]).min
    spots, last = [], []
    for row, length, n in zip(b.table_host, lens, news):
        hidden = list(range(sinks, max(sinks, length - n - window + 1))) + list(range(length, -(-length // page) * page))
        spots += [R.table_rows(row, page, b.pages, j) for j in hidden]
        last.append(R.table_rows(row, page, b.pages, length - 1))
    for t, at in ((b.kc, spots), (b.vc, spots), (b.vc, last)):
        pid, off = torch.tensor(at).T.cuda()
        t[pid, :, off] = value
    out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
    out, ref = out.double().cpu().numpy(), attention(b, window=window, sinks=sinks)
    last = np.array(b.starts[1:]) - 1
    others = np.setdiff1d(np.arange(b.starts[-1]), last)
    if others.size:
        assert np.abs(out[others] - ref[others]).max() <= TOL[dtype] * 6  # (|v| < 6)
    if not np.isfinite(value):  # the last rows: the formula's infinities and NaN
        assert np.array_equal(out[last], ref[last], equal_nan=True)


@gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("page", [32, 40])
@pytest.mark.parametrize("route", list(ROUTES))
def test_routes_with_rows_that_see_nothing(route, page, dtype):
    """Pages that are gone, sequences shorter than their new rows, and rows behind the last sequence."""
    from nkilab import ops

    b = batch(route, dtype, 64, page, seed=43)
    news = ROUTES[route][1]
    gone = len(news) - 1
    b.table_host[gone] = [b.pages + 5 if i % 2 else -1 for i in range(len(b.table_host[gone]))]
    if len(news) > 2:
        b.lens_host[1] = news[1] // 2  # (its first new rows have no place)
    table = torch.tensor(b.table_host, dtype=torch.int32).cuda()
    lens = torch.tensor(b.lens_host, dtype=torch.int32).cuda()
    q = torch.cat((b.q, b.q[:1].repeat(3, 1, 1)))
    o = torch.full_like(q, 7.0)
    ops.paged_attention_into(q, o, b.kc, b.vc, table, lens, q_start=b.q_start, max_q=b.max_q)
    check(b, o[:-3])
    assert (o[-3:] == 7).all() and not o[b.starts[gone]:b.starts[gone + 1]].any()
