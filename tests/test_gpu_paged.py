"""The paged cache's operators on the GPU against their definitions in 64 bits."""
import math
import random

import numpy as np
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# Attention outputs are weighted means of V, and weights sum to 1: an error of
# a relative e in every weight is at most e max|v| in the mean.  P and O are
# rounded by half a step each (eps / 2 of the type) in 16 bits; scores come of
# fp32 sums of d <= 128 products, and |s| <= |q| |k| scale < 16 for the inputs
# here: 128 roundings of 2^-24 on 16 are below 2^-13, which exp2 turns into a
# relative 2^-13 of a weight, twice (the mean's numerator and denominator).
TOL = {n: 2 * torch.finfo(t).eps / 2 * (0 if n == "fp32" else 1) + 2 * 2.0 ** -13 for n, t in DT.items()}


def close(out, ref, dtype, vmax):
    out = out.double().cpu().numpy()
    assert out.shape == ref.shape
    err = np.abs(out - ref).max() if out.size else 0.0
    assert err <= TOL[dtype] * vmax, (dtype, err, TOL[dtype] * vmax)


class Batch:
    """A random cache with its sequences, and their new rows."""

    def __init__(self, seed, lens, news, H, Hkv, d, page, dtype, spare=2, layout="page_major"):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        need = [-(-length // page) for length in lens]
        self.pages = sum(need) + spare
        pool = list(range(self.pages))
        rng.shuffle(pool)
        width = max(need + [1])
        rows, at = [], 0
        for c in need:
            rows.append(pool[at:at + c] + [-1] * (width - c))
            at += c
        self.table_host = rows
        self.table = torch.tensor(rows, dtype=torch.int32).cuda()
        self.lens_host, self.lens = list(lens), torch.tensor(lens, dtype=torch.int32).cuda()
        self.starts = [0]
        for n in news:
            self.starts.append(self.starts[-1] + n)
        self.q_start = torch.tensor(self.starts, dtype=torch.int32).cuda()
        self.max_q = max(news + [0])
        T = self.starts[-1]
        shape = (self.pages, Hkv, page, d)
        r = lambda *s: torch.randn(*s, generator=g).to(DT[dtype]).cuda()  # noqa: E731
        self.kc, self.vc = r(*shape), r(*shape)
        if layout == "row_major":  # rows of every head together
            self.kc, self.vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (self.kc, self.vc))
        self.q = r(T, H, d)
        self.dtype, self.page, self.H, self.Hkv, self.d = dtype, page, H, Hkv, d

    def args(self):
        return self.kc, self.vc, self.table, self.lens

    def ref(self, **kw):
        return R.attention(self.q.float().cpu(), self.kc.float().cpu(), self.vc.float().cpu(), self.table_host,
                           self.lens_host, self.starts, **kw)

    def check(self, out, **kw):
        vmax = float(self.vc.float().abs().max())
        close(out, self.ref(**kw), self.dtype, vmax)


# lens, news, H, Hkv, d, page
SHAPES = [
    ([1], [1], 1, 1, 64, 16),                       # one token, one key
    ([33, 1, 70], [1, 1, 1], 8, 2, 128, 16),        # single tokens, grouped heads
    ([40, 300, 5], [5, 130, 5], 4, 4, 128, 64),     # chunks; a whole prompt of 5
    ([65, 129], [33, 64], 6, 2, 32, 24),            # pages that end inside a tile
    ([700, 31], [3, 2], 7, 1, 96, 100),             # one K/V head for all, an odd group
    ([257], [257], 2, 1, 64, 256),                  # a prompt over a page and one row
    ([2000], [1], 4, 4, 128, 32),                   # long enough to split
]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (40, 3), (64, 40), (10 ** 9, 5)])
def test_chunks(shape, dtype, window, sinks):
    from nkilab import ops

    b = Batch(1, *shape, dtype)
    out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
    b.check(out, window=window, sinks=sinks)


def parents_of(rng, n, kind):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1] * n
    return [-1] + [rng.randrange(max(0, i - 9), i) for i in range(1, n)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lens,news,H,Hkv,d,page", [
    ([20], [20], 2, 2, 64, 16),                     # no context
    ([45, 100, 8], [16, 7, 1], 8, 2, 128, 16),
    ([130, 71], [70, 64], 4, 1, 128, 64),           # past a mask word
    ([333, 500], [150, 3], 3, 3, 64, 24),
    ([1500], [16], 4, 4, 128, 64),
], ids=str)
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "tree"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 4)])
def test_trees(lens, news, H, Hkv, d, page, dtype, kind, window, sinks):
    from nkilab import ops

    b = Batch(2, lens, news, H, Hkv, d, page, dtype)
    rng = random.Random(3)
    parents = [parents_of(rng, n, kind) for n in news]
    flat = torch.tensor(sum(parents, []), dtype=torch.int32).cuda()
    tree = ops.tree_mask(flat, q_start=b.q_start, max_q=b.max_q)
    bits = sum((R.tree_bits(p) for p in parents), [])
    width = tree.shape[1]
    for t, row in enumerate(bits):
        words = [sum(bit << i for i, bit in enumerate(row[64 * w:64 * w + 64])) for w in range(width)]
        assert [x % 2 ** 64 for x in tree[t].tolist()] == words
    out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, tree=tree, window=window, sinks=sinks)
    b.check(out, window=window, sinks=sinks, bits=bits)
    if kind == "chain" and (window or 10 ** 9) >= max(news):  # a chain is a prompt chunk (nodes: by their bits alone)
        same = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
        err = float((out.float() - same.float()).abs().max())
        assert err <= 2 * TOL[dtype] * float(b.vc.float().abs().max())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H,Hkv,S,d", [(2, 2, 1, 64), (4, 2, 200, 64), (1, 1, 300, 128), (6, 2, 515, 40), (2, 1, 257, 20)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (32, 0), (33, 5), (100, 64), (1000, 2)])
def test_window_prompts(H, Hkv, S, d, dtype, window, sinks):
    from nkilab import ops

    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(h, S, d, generator=g).to(DT[dtype]).cuda() for h in (H, Hkv, Hkv))
    out = ops.attention(q, k, v, window=window, sinks=sinks)
    kc, vc = (t.float().cpu()[None] for t in (k, v))
    ref = R.attention(q.float().cpu().transpose(0, 1), kc, vc, [[0]], [S], [0, S], window=window, sinks=sinks)
    close(out.transpose(0, 1), ref, dtype, float(v.float().abs().max()))


# ------------------------------------------------- what is masked or missing --

def poison(b, value):
    """Every K and V row that no sequence holds becomes `value`."""
    held = torch.zeros(b.pages, b.page, dtype=torch.bool)
    for row, length in zip(b.table_host, b.lens_host):
        for j in range(length):
            spot = R.table_rows(row, b.page, b.pages, j)
            if spot:
                held[spot] = True
    for t in (b.kc, b.vc):
        t.masked_fill_(~held.cuda()[:, None, :, None], value)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_rows_behind_a_sequence_may_hold_anything(dtype, value):
    from nkilab import ops

    b = Batch(5, [33, 100, 9], [1, 40, 9], 4, 2, 64, 24, dtype)
    poison(b, value)
    for window, sinks in ((None, 0), (30, 2)):
        out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
        ref = R.attention(b.q.float().cpu(), b.kc.float().cpu(), b.vc.float().cpu(), b.table_host, b.lens_host, b.starts,
                          window=window, sinks=sinks)
        assert np.isfinite(ref).all()
        close(out, ref, dtype, 5.0)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["k", "v", "kv"])
@pytest.mark.parametrize("mode", ["chunk", "window", "tree"])
def test_masked_keys_take_no_part(dtype, value, where, mode):
    """A key that some rows of a tile see and others do not: only those that see
    it know of it (V: what the formula gives; K: NaN rows)."""
    from nkilab import ops

    b = Batch(6, [90, 41], [30, 12], 4, 2, 64, 16, dtype)
    spot = R.table_rows(b.table_host[0], b.page, b.pages, 75)  # new row 15 of sequence 0
    if "k" in where:
        b.kc[spot[0], 1, spot[1]] = value
    if "v" in where:
        b.vc[spot[0], 1, spot[1], 5:9] = value
    kw = dict(window=10, sinks=1) if mode == "window" else {}
    tree = bits = None
    if mode == "tree":
        parents = [[-1] + [0] * 29, [-1] + [0] * 11]
        tree = ops.tree_mask(torch.tensor(sum(parents, []), dtype=torch.int32).cuda(), q_start=b.q_start, max_q=b.max_q)
        bits = sum((R.tree_bits(p) for p in parents), [])
    out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, tree=tree, **kw).double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        ref = b.ref(bits=bits, **kw)
    saw = [R.sees(i, 75, 30, 90, kw.get("window"), kw.get("sinks", 0), None if bits is None else bits[i])
           for i in range(30)] + [False] * 12
    assert any(saw) and not all(saw[:30])
    for t, s in enumerate(saw):
        for h in range(4):
            if s and h >= 2:
                if where == "v":  # finite columns as ever, the others as the formula has them
                    hit = np.zeros(64, bool)
                    hit[5:9] = True
                    assert np.array_equal(out[t, h][hit], ref[t, h][hit], equal_nan=True)
                    assert np.abs(out[t, h] - ref[t, h])[~hit].max() <= TOL[dtype] * 5
            else:
                assert np.abs(out[t, h] - ref[t, h]).max() <= TOL[dtype] * 5, (t, h)


@pytest.mark.parametrize("dtype", list(DT))
def test_freed_and_bad_pages(dtype):
    """Pages outside every row's window are not looked at; entries that name no
    page hold no keys; a row that sees nothing gets zeros."""
    from nkilab import ops

    b = Batch(7, [300, 64, 50], [1, 1, 2], 4, 2, 64, 16, dtype)
    kw = dict(q_start=b.q_start, max_q=b.max_q)
    before = ops.paged_attention(b.q, *b.args(), window=40, sinks=3, **kw)
    freed = b.table.clone()
    freed[0, 1:16] = -7  # of sequence 0, rows 16 .. 255: its window starts at 260
    after = ops.paged_attention(b.q, b.kc, b.vc, freed, b.lens, window=40, sinks=3, **kw)
    assert torch.equal(before, after)
    b.table_host = [list(r) for r in b.table_host]
    b.table_host[0][3], b.table_host[0][18] = b.pages, 2 ** 31 - 1
    b.table_host[1] = [-1] * len(b.table_host[1])
    b.table = torch.tensor(b.table_host, dtype=torch.int32).cuda()
    out = ops.paged_attention(b.q, *b.args(), **kw)
    b.check(out)
    assert not out[1].any()


def test_empty_and_short_sequences():
    """Lengths of zero, new rows that no length covers, lengths past the table."""
    from nkilab import ops

    b = Batch(8, [20, 37, 12, 80], [4, 3, 12, 2], 2, 2, 64, 16, "fp32")
    b.lens_host[0], b.lens_host[1], b.lens_host[2] = 0, 1, 5
    b.lens = torch.tensor(b.lens_host, dtype=torch.int32).cuda()
    out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q)
    b.check(out)
    assert not out[:4].any() and not out[4:6].any() and out[6].any()
    cut = b.table[:, :2].contiguous()  # 32 rows of each
    b.lens_host = [20, 37, 12, 80]
    b.lens = torch.tensor(b.lens_host, dtype=torch.int32).cuda()
    b.table_host = [r[:2] for r in b.table_host]
    out = ops.paged_attention(b.q, b.kc, b.vc, cut, b.lens, q_start=b.q_start, max_q=b.max_q)
    b.check(out)


def test_rows_of_no_sequence_are_left_alone():
    from nkilab import ops

    b = Batch(9, [50, 30], [3, 2], 4, 4, 64, 16, "bf16")
    q = torch.cat((b.q, b.q[:3]))
    out = torch.full_like(q, 7.0)
    ops.paged_attention_into(q, out, *b.args(), q_start=b.q_start, max_q=b.max_q)
    assert (out[5:] == 7).all()
    b.check(out[:5])
    out = torch.full_like(q, 7.0)  # only two new rows of a sequence are asked for
    ops.paged_attention_into(q, out, *b.args(), q_start=b.q_start, max_q=2)
    assert (out[2] == 7).all() and (out[5:] == 7).all()
    ref = b.ref()
    close(out[[0, 1, 3, 4]], ref[[0, 1, 3, 4]], "bf16", 5.0)
    # offsets out of order or out of range hold no rows
    bad = torch.tensor([4, 1, 99], dtype=torch.int32).cuda()
    out = torch.full_like(q, 7.0)
    ops.paged_attention_into(q, out, *b.args(), q_start=bad, max_q=8)
    assert (out[:1] == 7).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_strides(dtype):
    """Caches whose heads lie together, q and o as columns of wider rows, a table with spare columns."""
    from nkilab import ops

    for lens, news in (([200, 33], [1, 1]), ([200, 90], [70, 40])):
        b = Batch(10, lens, news, 6, 2, 64, 16, dtype, layout="row_major")
        T = b.q.shape[0]
        wide = torch.randn(T, 3, 6, 80, device="cuda").to(DT[dtype])
        wide[:, 1, :, :64] = b.q
        q = wide[:, 1, :, :64]
        o = torch.zeros(T, 7, 6, 64, dtype=DT[dtype], device="cuda")
        table = torch.cat((b.table, b.table.flip(0)), dim=1)[:, :b.table.shape[1]]
        ops.paged_attention_into(q, o[:, 2], b.kc, b.vc, table, b.lens, q_start=b.q_start, max_q=b.max_q)
        b.check(o[:, 2])
        assert not o[:, :2].any() and not o[:, 3:].any()
        # rows that are not on 16 bytes are copied first
        odd = torch.zeros(T, 6, 65, dtype=DT[dtype], device="cuda")
        odd[:, :, 1:] = b.q
        o2 = torch.zeros(T, 6, 67, dtype=DT[dtype], device="cuda")
        ops.paged_attention_into(odd[:, :, 1:], o2[:, :, 2:66], *b.args(), q_start=b.q_start, max_q=b.max_q)
        b.check(o2[:, :, 2:66])
        assert not o2[:, :, :2].any() and not o2[:, :, 66:].any()


def test_uniform_rows_need_no_offsets():
    from nkilab import ops

    b = Batch(11, [50, 30, 61], [2, 2, 2], 4, 4, 64, 16, "fp16")
    b.check(ops.paged_attention(b.q, *b.args()))


def test_offsets_past_32_bits():
    """Pages, rows and heads whose byte offsets do not fit 32 bits."""
    from nkilab import ops

    pages, page, d = 70000, 64, 128  # 9.2 GB each of K and V with two heads
    kc = torch.empty(pages, 2, page, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    ids = [69999, 3, 40000, 65536, 32768]
    b = Batch(12, [300], [2], 4, 2, d, page, "bf16")
    for i, src in zip(ids, b.table_host[0]):
        kc[i], vc[i] = b.kc[src], b.vc[src]
    table = torch.tensor([ids], dtype=torch.int32).cuda()
    b.check(ops.paged_attention(b.q, kc, vc, table, b.lens))
    # and the movers
    new = torch.randn(2, 2, d, device="cuda").bfloat16()
    ops.cache_append_into(new, new, kc, vc, table, b.lens)
    assert torch.equal(kc[32768, :, 42:44].transpose(0, 1), new) and torch.equal(vc[32768, :, 42:44].transpose(0, 1), new)
    ops.cache_copy_pages(kc, vc, [(69999, 69000), (3, 69998)])
    assert torch.equal(kc[69000], kc[69999]) and torch.equal(vc[69998], vc[3])
    k1 = kc[32768, :, 43].clone()
    ops.cache_accept(kc, vc, table, b.lens, torch.tensor([[1]], dtype=torch.int32).cuda(), n_nodes=2)
    assert torch.equal(kc[32768, :, 42], k1)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lens,news,H,Hkv", [
    ([5000, 17, 1], [1, 1, 1], 8, 2), ([40, 3000], [1, 64], 8, 2), ([2600] * 3, [70] * 3, 4, 4), ([1200] * 70, [1] * 70, 1, 1),
], ids=str)
def test_split_keys(dtype, lens, news, H, Hkv):
    """Long sequences beside short ones, keys split over workgroups; the same bits every time."""
    from nkilab import ops

    b = Batch(13, lens, news, H, Hkv, 64, 64, dtype)
    for window, sinks in ((None, 0), (2000, 70)):
        kw = dict(q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
        out = ops.paged_attention(b.q, *b.args(), **kw)
        b.check(out, window=window, sinks=sinks)
        assert torch.equal(out, ops.paged_attention(b.q, *b.args(), **kw))


def test_large_scores():
    """Scores far apart, and a running maximum that climbs with every tile."""
    from nkilab import ops

    b = Batch(14, [400], [3], 2, 2, 64, 16, "fp32")
    ramp = torch.linspace(-30, 30, 400).cuda()
    for j in range(400):
        p, o = R.table_rows(b.table_host[0], b.page, b.pages, j)
        b.kc[p, :, o] = ramp[j] * b.q[0, 0] / 8
    out = ops.paged_attention(b.q, *b.args(), scale=1.0)
    # |s| up to 30/8 |q|^2, near 300: 20 times the scores that TOL counts on
    ref = b.ref(scale=1.0)
    err = np.abs(out.double().cpu().numpy() - ref).max()
    assert err <= 20 * TOL["fp32"] * 5, err


# ----------------------------------------------- streams, graphs and threads --

def step_inputs(dtype="bf16"):
    return Batch(15, [900, 333, 40], [1, 1, 1], 8, 2, 64, 16, dtype)


def test_other_stream():
    from nkilab import ops

    b = step_inputs()
    want = ops.paged_attention(b.q, *b.args())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.paged_attention(b.q, *b.args()) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)


def test_captured_step_replays_with_other_lengths():
    """Append, attention and accept in one graph: replayed with other rows,
    lengths and tables beside eager work, each replay against the eager call."""
    from nkilab import ops

    b = Batch(16, [1200, 333, 64], [4, 4, 4], 8, 2, 64, 16, "bf16")
    T = 12
    k, v, q = (torch.randn(T, h, 64, device="cuda").bfloat16() for h in (2, 2, 8))
    q_rot = torch.empty_like(q)
    paths = torch.tensor([[0, 2, 3], [1, 3, -1], [-1, -1, -1]], dtype=torch.int32).cuda()
    parents = torch.tensor([-1, 0, 0, 2] * 3, dtype=torch.int32).cuda()

    def step(kc, vc):
        tree = ops.tree_mask(parents, batch=3)
        ops.cache_append_into(k, v, kc, vc, b.table, b.lens, tree=tree, q=q, q_out=q_rot, rope_base=10000.0)
        o = ops.paged_attention(q_rot, kc, vc, b.table, b.lens, tree=tree)
        return o, ops.cache_accept(kc, vc, b.table, b.lens, paths, n_nodes=4)

    kc, vc = b.kc.clone(), b.vc.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(kc, vc)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same call share nothing that they write
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(kc, vc)
        graphs.append((g, outs))
    for i, lens in enumerate(([1200, 333, 64], [1100, 40, 4], [17, 332, 60], [1196, 9, 33])):
        b.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        k.normal_(), v.normal_(), q.normal_()
        kc.copy_(b.kc), vc.copy_(b.vc)
        o, new = step(kc, vc)
        o, new, want_k, want_v = o.clone(), new.clone(), kc.clone(), vc.clone()
        kc.copy_(b.kc), vc.copy_(b.vc)
        torch.cuda.synchronize()
        g, (go, gnew) = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(go, o) and torch.equal(gnew, new) and torch.equal(kc, want_k) and torch.equal(vc, want_v)


# ------------------------------------------------------------------ append --

def rope_close(out, ref, dtype, xmax):
    """One rounding of the result (half a step), sine and cosine in 32 bits
    from an angle of at most pi (error below 2^-21) and three roundings of 2^-24."""
    half = torch.finfo(DT[dtype]).eps / 2 if dtype != "fp32" else 0.0
    err = np.abs(out.double().cpu().numpy() - ref)
    bound = half * np.abs(ref) + (2.0 ** -21 + 3 * 2.0 ** -24) * 2 * xmax + 2.0 ** -24
    assert (err <= bound).all(), float((err - bound).max())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("base", [None, 10000.0, 500000.0])
@pytest.mark.parametrize("lens,news,H,Hkv,d,page", [
    ([1], [1], 1, 1, 64, 16),
    ([33, 1, 70, 5], [1, 1, 1, 0], 8, 2, 128, 16),
    ([40, 300], [40, 130], 4, 4, 96, 64),
    ([25, 9], [20, 9], 3, 1, 20, 24),               # rows off 16 bytes
    ([700] * 40, [60] * 40, 2, 2, 32, 100),
], ids=str)
def test_append(lens, news, H, Hkv, d, page, dtype, base):
    from nkilab import ops

    b = Batch(17, lens, news, H, Hkv, d, page, dtype)
    T = b.starts[-1]
    # k and v as columns of packed projections
    packed = torch.randn(T, H + 2 * Hkv, d, device="cuda").to(DT[dtype])
    q, k, v = packed[:, :H], packed[:, H:H + Hkv], packed[:, H + Hkv:]
    q_host, k_host, v_host = (t.float().cpu().numpy() for t in (q, k, v))
    want_k, want_v = b.kc.double().cpu().numpy(), b.vc.double().cpu().numpy()
    kw = {}
    if base:
        kw = dict(q=q, q_out=q, rope_base=base)  # in place
    ops.cache_append_into(k, v, *b.args(), q_start=b.q_start, max_q=b.max_q, **kw)
    want_q = np.array(q_host, np.float64)
    for s, length in enumerate(lens):
        for i in range(news[s]):
            t, pos = b.starts[s] + i, length - news[s] + i
            p, o = R.table_rows(b.table_host[s], page, b.pages, pos)
            want_k[p, :, o] = R.rope(k_host[t], pos, base) if base else k_host[t]
            want_v[p, :, o] = v_host[t]
            if base:
                want_q[t] = R.rope(q_host[t], pos, base)
    xmax = float(packed.float().abs().max()) + 5
    assert np.array_equal(b.vc.double().cpu().numpy(), want_v)
    if base:
        rope_close(b.kc, want_k, dtype, xmax)
        rope_close(q, want_q, dtype, xmax)
    else:
        assert np.array_equal(b.kc.double().cpu().numpy(), want_k)
    assert torch.equal(k.float().cpu(), torch.from_numpy(k_host))


def test_append_rotates_a_tree_by_depth():
    from nkilab import ops

    b = Batch(18, [40, 80], [6, 70], 2, 1, 64, 16, "fp32")
    rng = random.Random(1)
    parents = [parents_of(rng, n, "tree") for n in (6, 70)]
    tree = ops.tree_mask(torch.tensor(sum(parents, []), dtype=torch.int32).cuda(), q_start=b.q_start, max_q=b.max_q)
    k, v = (torch.randn(76, 1, 64, device="cuda") for _ in range(2))
    q_out = torch.empty_like(b.q)
    ops.cache_append_into(k, v, *b.args(), q_start=b.q_start, max_q=b.max_q, tree=tree, q=b.q, q_out=q_out,
                          rope_base=10000.0)
    want = np.zeros((76, 2, 64))
    for s, (length, n) in enumerate(zip([40, 80], [6, 70])):
        bits = R.tree_bits(parents[s])
        for i in range(n):
            t, pos = b.starts[s] + i, length - n + sum(bits[i]) - 1
            want[t] = R.rope(b.q[t].cpu().numpy(), pos, 10000.0)
            p, o = R.table_rows(b.table_host[s], 16, b.pages, length - n + i)
            rope_close(b.kc[p, :, o], R.rope(k[t].cpu().numpy(), pos, 10000.0), "fp32", 6)
    rope_close(q_out, want, "fp32", 6)


@pytest.mark.parametrize("dtype", list(DT))
def test_append_far_positions(dtype):
    """Angles of positions that 32 bits cannot hold to a radian."""
    from nkilab import ops

    page, cols = 1 << 16, 400
    length = page * cols - 5  # above 2^24
    kc = torch.zeros(1, 1, page, 32, dtype=DT[dtype], device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.full((1, cols), -1, dtype=torch.int32, device="cuda")
    table[0, cols - 1] = 0
    x = torch.randn(3, 1, 32, device="cuda").to(DT[dtype])
    ops.cache_append_into(x, x, kc, vc, table, torch.tensor([length], dtype=torch.int32).cuda(), rope_base=10000.0)
    ref = np.stack([R.rope(x[i].float().cpu().numpy(), length - 3 + i, 10000.0) for i in range(3)])
    at = page - 5 - 3
    rope_close(kc[0, :, at:at + 3].transpose(0, 1), ref, dtype, 5)
    assert torch.equal(vc[0, :, at:at + 3].transpose(0, 1), x)
    assert int((vc != 0).any(dim=-1).sum()) == 3


def test_append_skips_rows_without_a_place():
    from nkilab import ops

    b = Batch(19, [40, 30, 20], [4, 4, 4], 2, 2, 64, 16, "fp32")
    table = b.table.clone()
    table[0, 2] = -1                       # sequence 0: rows 32 .. 47 have no page
    table[1, 1] = b.pages                  # sequence 1: rows 16 .. 31 neither
    lens = torch.tensor([40, 30, 2], dtype=torch.int32).cuda()  # sequence 2: two rows at negative positions
    k, v = (torch.randn(15, 2, 64, device="cuda") for _ in range(2))
    kc, vc = b.kc.clone(), b.vc.clone()
    ops.cache_append_into(k, v, kc, vc, table, lens, q_start=b.q_start, max_q=4)  # 3 rows of no sequence
    changed = (vc != b.vc).any(dim=-1).any(dim=1)
    p = b.table_host[2][0]
    assert changed.nonzero().tolist() == [[p, 0], [p, 1]]
    assert torch.equal(vc[p, :, :2].transpose(0, 1), v[10:12]) and torch.equal(kc[p, :, :2].transpose(0, 1), k[10:12])


# ---------------------------------------------------------- pages and paths --

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape,layout", [
    ((5, 2, 16, 64), "plain"), ((3, 700, 2, 8, 32), "plain"), ((2, 9, 3, 24, 20), "plain"), ((6, 4, 16, 64), "row_major"),
    ((2, 6, 2, 7, 3), "plain"), ((3, 6, 2, 256, 128), "layers_last"),
], ids=str)
def test_copy_pages(shape, layout, dtype):
    from nkilab import ops

    kc, vc = (torch.randn(*shape, device="cuda").to(DT[dtype]) for _ in range(2))
    if layout == "row_major":
        kc, vc = (t.transpose(-3, -2).contiguous().transpose(-3, -2) for t in (kc, vc))
    if layout == "layers_last":  # pages outermost, and v laid out unlike k
        kc = kc.transpose(0, 1).contiguous().transpose(0, 1)
    pages = shape[-4]
    ids = list(range(pages))
    random.Random(2).shuffle(ids)
    pairs = list(zip(ids[: pages // 2], ids[pages // 2:]))
    want = [t.clone() for t in (kc, vc)]
    for w in want:
        w5 = w if w.dim() == 5 else w[None]
        for a, z in pairs:
            w5[:, z] = w5[:, a]
    ops.cache_copy_pages(kc, vc, np.array(pairs))
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    for w in want:  # one source, several copies
        w5 = w if w.dim() == 5 else w[None]
        for z in ids[1:4]:
            w5[:, z] = w5[:, ids[0]]
    ops.cache_copy_pages(kc, vc, [(ids[0], z) for z in ids[1:4]])
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def accept_reference(kc, vc, table_host, lens, news, paths, page):
    """Every row read before any is written; the path ends at its first entry that does not ascend within [0, n)."""
    pages = kc.shape[-4]
    new = []
    for b, path in enumerate(paths):
        n, ctx = news[b], lens[b] - news[b]
        kept = []
        for node in path:
            if not (kept[-1] if kept else -1) < node < n:
                break
            kept.append(node)
        new.append(max(0, ctx + len(kept)))
        for t in (kc, vc):
            old = t.clone()
            for i, node in enumerate(kept):
                src, dst = (R.table_rows(table_host[b], page, pages, ctx + r) for r in (node, i))
                if src and dst:
                    t[..., dst[0], :, dst[1], :] = old[..., src[0], :, src[1], :]
    return new


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("layers,d,page,layout", [(None, 64, 16, "plain"), (3, 128, 24, "plain"), (2, 20, 8, "plain"),
                                                  (None, 32, 16, "row_major")])
def test_accept(dtype, layers, d, page, layout):
    from nkilab import ops

    news = [16, 300, 5, 7, 4, 3, 40]
    lens = [100, 301, 5, 30, 2, 50, 40]  # (the fifth is shorter than its nodes)
    b = Batch(20, [max(n, x) for n, x in zip(lens, news)], news, 1, 3, d, page, dtype, layout=layout)
    if layers:
        b.kc, b.vc = (torch.stack([t + i for i in range(layers)]) for t in (b.kc, b.vc))
    paths = [[2, 3, 5, 9, 15],              # rows that are read again further on
             list(range(1, 299)),           # longer than a batch of entries, every row one down
             [0, 1, 2, 3, 4],               # in place
             [3, 3, 5],                     # ends where it does not ascend
             [1, 2, 3],
             [2, 3],                        # ends past the nodes
             []]
    width = max(map(len, paths))
    table = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32).cuda()
    want_k, want_v = b.kc.cpu().clone(), b.vc.cpu().clone()
    new = accept_reference(want_k, want_v, b.table_host, lens, news, paths, page)
    got = ops.cache_accept(b.kc, b.vc, b.table, torch.tensor(lens, dtype=torch.int32).cuda(), table, q_start=b.q_start)
    assert got.tolist() == new == [89, 299, 5, 24, 1, 48, 0]
    assert torch.equal(b.kc.cpu(), want_k) and torch.equal(b.vc.cpu(), want_v)


def test_accept_of_nothing():
    from nkilab import ops

    b = Batch(21, [30, 30], [4, 4], 1, 1, 64, 16, "bf16")
    before = b.kc.clone()
    none = torch.empty(2, 0, dtype=torch.int32).cuda()
    assert ops.cache_accept(*b.args(), none, n_nodes=4).tolist() == [26, 26]
    assert ops.cache_accept(*b.args(), torch.tensor([[0, 9], [-1, 2]], dtype=torch.int32).cuda(), n_nodes=4).tolist() == \
        [27, 26]
    assert torch.equal(b.kc, before)


def test_tree_mask_ends_at_bad_parents():
    """A parent that is not below its node is none; rows of no tree see nothing."""
    from nkilab import ops

    parents = torch.tensor([-1, 0, 5, 3, 2, -1, 0, 9, 9], dtype=torch.int32).cuda()
    q_start = torch.tensor([0, 5, 7], dtype=torch.int32).cuda()
    m = ops.tree_mask(parents, q_start=q_start, max_q=5)
    assert m[:, 0].tolist() == [0b1, 0b11, 0b100, 0b1000, 0b10100, 0b1, 0b11, 0, 0]
    chain = torch.arange(-1, 4999, dtype=torch.int32).cuda()  # past the nodes held on the chip
    m = ops.tree_mask(chain)
    assert m.shape == (5000, 79)
    pop = torch.tensor([[bin(w % 2 ** 64).count("1") for w in r] for r in m[::499].tolist()]).sum(dim=1)
    assert pop.tolist() == [i + 1 for i in range(0, 5000, 499)]


# ------------------------------------------------------------- odd batches --

@pytest.mark.parametrize("dtype", list(DT))
def test_one_prompt_among_single_tokens(dtype):
    """Sequences whose new rows differ a hundredfold, more of them than a wavefront has lanes."""
    from nkilab import ops

    news = [1] * 40 + [150] + [0] + [1] * 60
    lens = [5 + 3 * i for i in range(40)] + [170] + [7] + [1 + i for i in range(60)]
    b = Batch(22, lens, news, 4, 2, 64, 16, dtype)
    for window, sinks in ((None, 0), (50, 2)):
        out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
        b.check(out, window=window, sinks=sinks)


@pytest.mark.parametrize("batch", [1, 63, 64, 65, 200, 4100])
def test_append_of_one_prompt_among_single_tokens(batch):
    """Rows placed by a search over the offsets, empty sequences among them."""
    from nkilab import ops

    rng = random.Random(batch)
    news = [rng.choice((0, 1, 1, 2)) for _ in range(batch)]
    news[batch // 2] = 700
    lens = [n + rng.randint(0, 3) for n in news]
    b = Batch(23, lens, news, 1, 1, 32, 16, "fp32")
    T = b.starts[-1]
    k, v = (torch.randn(T + 3, 1, 32, device="cuda") for _ in range(2))  # 3 rows of no sequence
    want_k, want_v = b.kc.cpu().clone(), b.vc.cpu().clone()
    for s in range(batch):
        for i in range(news[s]):
            p, o = R.table_rows(b.table_host[s], 16, b.pages, lens[s] - news[s] + i)
            want_k[p, :, o], want_v[p, :, o] = k[b.starts[s] + i].cpu(), v[b.starts[s] + i].cpu()
    ops.cache_append_into(k, v, *b.args(), q_start=b.q_start, max_q=b.max_q)
    assert torch.equal(b.kc.cpu(), want_k) and torch.equal(b.vc.cpu(), want_v)


@pytest.mark.parametrize("dtype", list(DT))
def test_nothing_to_do(dtype):
    """No sequences, no rows, no columns, no pages."""
    from nkilab import ops

    dt = DT[dtype]
    i32 = dict(dtype=torch.int32, device="cuda")
    kc, vc = (torch.randn(4, 2, 16, 64, device="cuda").to(dt) for _ in range(2))
    none = torch.empty(0, 2, 64, dtype=dt, device="cuda")
    table0, lens0 = torch.empty(0, 3, **i32), torch.empty(0, **i32)
    assert ops.paged_attention(none, kc, vc, table0, lens0).shape == (0, 2, 64)
    assert ops.paged_attention(none, kc, vc, table0, lens0, q_start=torch.zeros(1, **i32), max_q=0).shape == (0, 2, 64)
    ops.cache_append_into(none, none, kc, vc, table0, lens0)
    assert ops.cache_accept(kc, vc, table0, lens0, torch.empty(0, 2, **i32), n_nodes=3).shape == (0,)
    assert ops.tree_mask(torch.empty(0, **i32), batch=2).shape == (0, 1)
    q = torch.randn(2, 4, 64, device="cuda").to(dt)
    lens = torch.tensor([9, 3], **i32)
    # a table of no columns, and a cache of no pages, hold no keys
    assert not ops.paged_attention(q, kc, vc, torch.empty(2, 0, **i32), lens).any()
    assert not ops.paged_attention(q, kc[:0], vc[:0], torch.zeros(2, 3, **i32), lens).any()
    many = torch.randn(200, 4, 64, device="cuda").to(dt)
    assert not ops.paged_attention(many, kc[:0], vc[:0], torch.zeros(2, 300, **i32), lens).any()
    before = kc.clone()
    ops.cache_append_into(q[:, :2], q[:, :2], kc, vc, torch.empty(2, 0, **i32), lens)
    ops.cache_append_into(q[:, :2], q[:, :2], kc[:0], vc[:0], torch.zeros(2, 3, **i32), lens)
    paths = torch.tensor([[1], [0]], **i32)
    assert ops.cache_accept(kc, vc, torch.empty(2, 0, **i32), lens, paths, n_nodes=2).tolist() == [8, 2]
    assert ops.cache_accept(kc[:0], vc[:0], torch.zeros(2, 3, **i32), lens, paths, n_nodes=2).tolist() == [8, 2]
    assert torch.equal(kc, before)
    assert ops.attention(none.transpose(0, 1), none.transpose(0, 1), none.transpose(0, 1), window=4).shape == (2, 0, 64)


@pytest.mark.parametrize("dtype", list(DT))
def test_output_over_the_queries(dtype):
    """o may be q: whole row tiles and split ones."""
    from nkilab import ops

    for lens, news in (([3000, 40], [1, 1]), ([900, 333], [200, 33])):
        b = Batch(24, lens, news, 8, 2, 64, 16, dtype)
        want = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q)
        got = b.q.clone()
        ops.paged_attention_into(got, got, *b.args(), q_start=b.q_start, max_q=b.max_q)
        assert torch.equal(got, want)


@pytest.mark.parametrize("page", [1, 8, 16, 48, 4096])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_page_sizes(page, dtype):
    """Pages of one row, smaller than a tile's half, of halves and tiles, and longer than the sequences."""
    from nkilab import ops

    for lens, news in (([300, 33, 64], [1, 1, 1]), ([170, 600], [70, 130])):
        b = Batch(25, lens, news, 6, 3, 128, page, dtype)
        for window, sinks in ((None, 0), (37, 20)):
            out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
            b.check(out, window=window, sinks=sinks)


@pytest.mark.parametrize("d", [8, 24, 40, 72, 104, 120])
@pytest.mark.parametrize("dtype", list(DT))
def test_head_dims(d, dtype):
    from nkilab import ops

    for lens, news in (([300, 33], [1, 1]), ([170, 90], [70, 5])):
        b = Batch(26, lens, news, 4, 2, d, 32, dtype)
        poison(b, float("nan"))
        out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q)
        ref = R.attention(b.q.float().cpu(), b.kc.float().cpu(), b.vc.float().cpu(), b.table_host, b.lens_host, b.starts)
        close(out, ref, dtype, 5.0)


@pytest.mark.parametrize("dtype", list(DT))
def test_infinities_in_split_keys(dtype):
    """V's infinities and NaN where keys are split over workgroups and pages are
    halves of tiles: the rows that see them have them, the others do not."""
    from nkilab import ops

    b = Batch(27, [2500, 2500], [3, 70], 4, 2, 64, 16, dtype)
    for s, j, col, value in ((0, 2497, 3, float("inf")), (0, 2498, 4, float("nan")), (1, 2460, 5, float("-inf")),
                             (1, 10, 6, float("inf"))):
        p, o = R.table_rows(b.table_host[s], 16, b.pages, j)
        b.vc[p, 0, o, col] = value
    for window, sinks in ((None, 0), (2000, 16)):
        out = ops.paged_attention(b.q, *b.args(), q_start=b.q_start, max_q=b.max_q, window=window, sinks=sinks)
        got = out.double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            ref = b.ref(window=window, sinks=sinks)
        bad = ~np.isfinite(ref)
        assert bad.any() and np.array_equal(got[bad], ref[bad], equal_nan=True)
        assert np.abs(got[~bad] - ref[~bad]).max() <= TOL[dtype] * 5


def test_all_scores_nan():
    """A row whose every visible score is NaN is NaN, also where one part of its keys has nothing else."""
    from nkilab import ops

    b = Batch(28, [2500], [2], 2, 1, 64, 16, "bf16")
    b.q[0] = float("nan")
    out = ops.paged_attention(b.q, *b.args())
    assert out[0].isnan().all() and out[1].isfinite().all()
    b.q[0] = 1.0
    p, o = R.table_rows(b.table_host[0], 16, b.pages, 5)
    b.kc[p, 0, o] = float("nan")
    assert ops.paged_attention(b.q, *b.args()).isnan().all()
    assert ops.paged_attention(b.q, *b.args(), window=2000).isfinite().all()


@pytest.mark.parametrize("page", [64, 8])
def test_offsets_past_4_gib(page):
    """Byte offsets past 32 bits and element offsets past 31, in both kinds of loads."""
    from nkilab import ops

    d = 128
    pages = 2 ** 32 // (2 * 2 * page * d) + 50  # two heads of bf16
    kc = torch.empty(pages, 2, page, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    for lens, news in (([3 * page], [2]), ([3 * page], [3 * page])):
        b = Batch(29, lens, news, 4 if news == [2] else 40, 2, d, page, "bf16")
        ids = [pages - 1, pages // 2 + 1, pages - 40]
        for i, src in zip(ids, b.table_host[0]):
            kc[i], vc[i] = b.kc[src], b.vc[src]
        table = torch.tensor([ids], dtype=torch.int32).cuda()
        b.check(ops.paged_attention(b.q, kc, vc, table, b.lens))
    new = torch.randn(2, 2, d, device="cuda").bfloat16()
    ops.cache_append_into(new, new, kc, vc, table, b.lens)
    at = page - 2
    assert torch.equal(kc[ids[2], :, at:].transpose(0, 1), new) and torch.equal(vc[ids[2], :, at:].transpose(0, 1), new)
    ops.cache_copy_pages(kc, vc, [(ids[2], 0), (5, ids[0])])
    assert torch.equal(kc[0], kc[ids[2]]) and torch.equal(vc[ids[0]], vc[5])
    ops.cache_accept(kc, vc, table, b.lens, torch.tensor([[1]], dtype=torch.int32).cuda(), n_nodes=2)
    assert torch.equal(vc[ids[2], :, at], new[1])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tree", [False, True])
def test_split_keys_of_many_sequences(dtype, tree):
    """More sequences than a wavefront has lanes, from no rows to long ones, in ranges over their keys."""
    from nkilab import ops

    lens = [(37 * i * i) % 2100 for i in range(70)]
    news = [min(n, 1 + i % 3) for i, n in enumerate(lens)]
    b = Batch(30, lens, news, 2, 1, 32, 32, dtype)
    kw, bits = dict(q_start=b.q_start, max_q=b.max_q, window=1500, sinks=33), None
    if tree:
        parents = [[-1, 0, 0][:n] for n in news]
        kw["tree"] = ops.tree_mask(torch.tensor(sum(parents, []), dtype=torch.int32).cuda(), q_start=b.q_start,
                                   max_q=b.max_q)
        bits = sum((R.tree_bits(p) for p in parents), [])
        bits = [row + [0] * (3 - len(row)) for row in bits]
    b.check(ops.paged_attention(b.q, *b.args(), **kw), window=1500, sinks=33, bits=bits)


@pytest.mark.parametrize("news", [1, 70])
def test_two_captured_graphs_share_no_workspace(news):
    """Calls whose keys are split, captured twice and replayed side by side on two
    streams, over lengths that change between replays."""
    from nkilab import ops

    first, second = (Batch(s, [6000, 300], [news] * 2, 4, 1, 64, 64, "bf16") for s in (31, 32))
    graphs = []
    for b in (first, second):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.paged_attention(b.q, *b.args())
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = ops.paged_attention(b.q, *b.args())
        graphs.append((g, s, out))
    for lens in ([6000, 300], [5000, 100], [news, 299], [3001, 256]):
        want = []
        for b in (first, second):
            b.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            want.append(ops.paged_attention(b.q, *b.args()))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s, _out in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for (_g, _s, out), w in zip(graphs, want):
            assert torch.equal(out, w)
    first.lens_host = lens
    first.check(graphs[0][2])
