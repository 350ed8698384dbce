"""Attention over the 8-bit paged cache on the GPU against its definition in 64 bits."""
import random

import numpy as np
import pytest
import torch

import cache8_reference as R8
import paged_reference as R
from test_gpu_cache8 import Cache

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# Outputs are weighted means of V, weights summing to 1: a relative error e in every weight is at most
# e max|v| in the mean.  P and O are rounded by half a step each in 16 bits (codes' values are exact, but for
# fp16 values below 2^-14, off by 2^-25 at most).  Scores are fp32 sums of d <= 128 products with |s| <= 16
# here: 128 roundings of 2^-24 on 16 are below 2^-13, a relative 2^-13 of a weight, twice (numerator and
# denominator).
TOL = {n: 2 * torch.finfo(t).eps / 2 * (0 if n == "fp32" else 1) + 2 * 2.0 ** -13 for n, t in DT.items()}


class Batch(Cache):
    """A cache of values of the order of one: codes of a normal distribution, pages of magnitudes up to four times apart."""

    def __init__(self, seed, lens, news, H, Hkv, d, page, dtype, layout="page_major"):
        super().__init__(seed, lens, Hkv, d, page, layout=layout)
        g = torch.Generator().manual_seed(seed + 1)
        for codes, scales in ((self.kc, self.ks), (self.vc, self.vs)):
            x = torch.randn(codes.shape, generator=g).clamp(-4, 4)
            codes.copy_((x * 100).to(torch.float8_e4m3fn).cuda())
            scales.copy_((119 + torch.randint(0, 3, scales.shape, generator=g)).to(torch.uint8))
        self.starts = [0] + [int(x) for x in np.cumsum(news)]
        self.q_start = torch.tensor(self.starts, dtype=torch.int32).cuda()
        self.max_q = max(news + [0])
        self.q = torch.randn(self.starts[-1], H, d, generator=g).to(DT[dtype]).cuda()
        self.dtype = dtype

    def call(self, **kw):
        from nkilab import ops

        kw.setdefault("q_start", self.q_start)
        return ops.paged_attention(self.q, self.kc, self.vc, self.table, self.lens, max_q=self.max_q, **kw, **self.scales())

    def ref(self, **kw):
        kc, ks, vc, vs = self.host()
        return R.attention(self.q.double().cpu().numpy(), R8.values(kc, ks), R8.values(vc, vs), self.table_host, self.lens_host,
                           self.starts, **kw)

    def check(self, out, **kw):
        want, out = self.ref(**kw), out.double().cpu().numpy()
        kc, ks, vc, vs = self.host()
        vmax = np.nanmax(np.abs(R8.values(vc, vs)))
        assert np.array_equal(np.isnan(out), np.isnan(want))
        err = np.nanmax(np.abs(out - want)) if out.size else 0.0
        assert err <= TOL[self.dtype] * vmax, (err, TOL[self.dtype] * vmax)


# lens, news, H, Hkv, d, page
SHAPES = [
    ([1], [1], 1, 1, 64, 16),                       # one token, one key
    ([33, 1, 70], [1, 1, 1], 8, 2, 128, 16),        # single tokens, grouped heads
    ([40, 300, 5], [5, 130, 5], 4, 4, 128, 64),     # chunks; a whole prompt of 5
    ([65, 129], [33, 64], 6, 2, 32, 24),            # pages that end inside a tile, narrow heads
    ([100, 37], [1, 1], 16, 2, 80, 100),            # a head dim between the tiles', pages off every tile
    ([900, 2100, 31], [1, 1, 1], 8, 8, 128, 64),    # keys split over workgroups
    ([700, 10], [2, 9], 14, 2, 64, 8),              # pages of half a half tile
    ([260], [260], 4, 1, 96, 32),                   # a prompt
    ([50, 600], [20, 600], 2, 2, 32, 16),           # narrow heads, more than 32 rows
    ([2300, 40], [70, 33], 4, 2, 64, 16),           # more key tiles than are looked up at a time
    ([2200], [40], 2, 1, 128, 32),
]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_attention8(shape, dtype):
    lens, news, H, Hkv, d, page = shape
    for i, layout in enumerate(("page_major", "row_major")):
        b = Batch(i, lens, news, H, Hkv, d, page, dtype, layout)
        b.check(b.call())
        for window, sinks in ((1, 0), (17, 3), (64, 0), (200, 40)):
            b.check(b.call(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DT)
def test_attention8_tree(dtype):
    from nkilab import ops

    rng = random.Random(3)
    for lens, news, H, Hkv, d, page in (([100, 64], [16, 64], 4, 2, 128, 16), ([1200], [100], 8, 2, 64, 24), ([20, 9], [3, 9], 16, 1, 32, 8)):
        b = Batch(5, lens, news, H, Hkv, d, page, dtype)
        parents = [p for n in news for p in [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)]]
        bits = [row for s, e in zip(b.starts, b.starts[1:]) for row in R.tree_bits(parents[s:e])]
        words = ops.tree_mask(torch.tensor(parents, dtype=torch.int32).cuda(), q_start=b.q_start, max_q=b.max_q)
        for window, sinks in ((None, 0), (30, 4)):
            b.check(b.call(tree=words, window=window, sinks=sinks), bits=bits, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DT)
def test_masked_nan_and_freed_pages(dtype):
    """NaN codes take no part where they are masked, and reach the rows that see them; pages that no row sees may name none;
    a row that sees nothing gets zeros."""
    lens, news, H, Hkv, d, page = [150, 90], [3, 40], 4, 2, 64, 16
    b = Batch(1, lens, news, H, Hkv, d, page, dtype)
    raw = lambda t: t.view(torch.uint8)  # noqa: E731
    for t in (b.kc, b.vc):
        raw(t)[b.table_host[0][2], 1, 5] = 127        # rows 37 and 149 of sequence 0
        raw(t)[b.table_host[0][9], 0, 5, 3] = 255
        raw(t)[b.table_host[1][5], :, 10:] = 127      # rows behind the last of sequence 1
    out = b.call(window=20)
    b.check(out, window=20)
    assert not torch.isnan(out[:2]).any() and torch.isnan(out[2, :2]).any() and not torch.isnan(out[3:]).any()
    b.check(b.call())
    b.table_host[0][:7] = [-1] * 7
    b.table_host[1][0], b.table_host[1][3] = b.pages, -5
    b.table = torch.tensor(b.table_host, dtype=torch.int32).cuda()
    b.check(b.call())
    b.check(b.call(window=9, sinks=2), window=9, sinks=2)
    b.table_host = [[-1] * len(r) for r in b.table_host]
    b.table = torch.tensor(b.table_host, dtype=torch.int32).cuda()
    assert not b.call().any()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("page", [16, 24])
def test_scales_far_apart(dtype, page):
    """Pages whose values differ by many powers of two, and magnitudes at the ends of the types."""
    b = Batch(2, [200], [4], 2, 1, 64, page, dtype)
    n = len(b.table_host[0])
    for i, p in enumerate(b.table_host[0]):
        b.vs[p] = 119 + (-14, 0, 6, -3)[i % 4]
        b.ks[p] = 119 - (0, 12, 1)[i % 3]
    b.check(b.call())
    # V as large as fp16 goes (65536 is not one of its numbers), or far beyond where the type has it
    big = {"fp16": 135, "bf16": 240, "fp32": 240}[dtype]
    raw = b.vc.view(torch.uint8)
    raw.copy_(torch.randint(0x70, 0x79, raw.shape, dtype=torch.uint8))
    b.vs.fill_(big)
    want = R.attention(b.q.double().cpu().numpy(), R8.values(*b.host()[:2]),
                       np.minimum(R8.values(*b.host()[2:]), 65504.0 if dtype == "fp16" else np.inf), b.table_host, b.lens_host, b.starts)
    out = b.call().double().cpu().numpy()
    assert np.isfinite(out).all() and (np.abs(out - want) <= TOL[dtype] * want.max()).all()
    # and as small
    b.vs.fill_({"fp16": 105, "bf16": 17, "fp32": 17}[dtype])
    want = b.ref()
    out = b.call().double().cpu().numpy()
    assert (np.abs(out - want) <= TOL[dtype] * want.max() + (2.0 ** -24 if dtype == "fp16" else 0)).all()
    assert n > 8


def test_rows_of_no_sequence_and_views():
    from nkilab import ops

    b = Batch(4, [40, 50], [2, 3], 4, 2, 64, 16, "bf16")
    q = torch.randn(9, 4, 64, device="cuda").bfloat16()
    q[:5] = b.q
    o = torch.full((9, 4, 70), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention_into(q, o[:, :, 6:], b.kc, b.vc, b.table, b.lens, q_start=b.q_start, max_q=3, **b.scales())
    assert (o[5:] == 3).all() and (o[:, :, :6] == 3).all()
    b.check(o[:5, :, 6:])


def test_streams_graphs_and_both_at_once():
    """Two captured calls with workspaces replayed side by side, with other lengths; the same results as one by one."""
    from nkilab import ops

    bs = [Batch(i, [900 + i, 2100, 31], [1, 1, 1], 8, 8, 128, 64, "bf16") for i in (1, 2)]
    outs = [torch.empty_like(b.q) for b in bs]
    run = lambda b, o: ops.paged_attention_into(b.q, o, b.kc, b.vc, b.table, b.lens, q_start=b.q_start, max_q=1, **b.scales())  # noqa: E731
    streams = [torch.cuda.Stream() for _ in bs]
    graphs = []
    for b, o, s in zip(bs, outs, streams):
        run(b, o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run(b, o)
        graphs.append(g)
    for lens in ([901, 2100, 31], [100, 1500, 30], [1, 64, 2]):
        for b in bs:
            b.lens_host = lens
            b.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b, o in zip(bs, outs):
            b.check(o)
            assert torch.equal(o, b.call())


def test_far_pages():
    """Pages more than 4 GiB into the cache."""
    from nkilab import ops

    pages, Hkv, page, d = (1 << 32) // (2 * 64 * 128) + 64, 2, 64, 128
    kc, vc = (torch.zeros(pages, Hkv, page, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((pages, Hkv), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(150, Hkv, d, generator=g).cuda() for _ in range(2))
    lens = torch.tensor([150], dtype=torch.int32, device="cuda")
    ops.cache_append_into(k, v, kc, vc, table, lens, k_scale=ks, v_scale=vs)
    q = torch.randn(150, 4, d, generator=g).cuda()
    o = ops.paged_attention(q, kc, vc, table, lens, k_scale=ks, v_scale=vs)
    # the same in a small cache
    pick = torch.tensor([pages - 1, 3, pages - 2], device="cuda")
    small = [t.view(torch.uint8)[pick].clone().view(torch.float8_e4m3fn) for t in (kc, vc)]
    near = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(o, ops.paged_attention(q, *small, near, lens, k_scale=ks[pick], v_scale=vs[pick]))
    assert o.abs().max() > 0.1 and torch.isfinite(o).all()
