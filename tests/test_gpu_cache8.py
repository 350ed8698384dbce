"""The 8-bit paged cache on the GPU: rows written (codes and scales have to be
equal to the definition's), pages copied, paths accepted."""
import random

import numpy as np
import pytest
import torch

import cache8_reference as R8

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


class Cache:
    """A random cache of codes and scales with its sequences' tables; layouts of the tensors vary."""

    def __init__(self, seed, lens, Hkv, d, page, spare=2, layout="page_major", lead=()):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        need = [-(-length // page) for length in lens]
        self.pages = sum(need) + spare
        pool = list(range(self.pages))
        rng.shuffle(pool)
        width, at, self.table_host = max(need + [1]), 0, []
        for c in need:
            self.table_host.append(pool[at:at + c] + [-1] * (width - c))
            at += c
        self.table = torch.tensor(self.table_host, dtype=torch.int32).view(len(lens), width).cuda()
        self.lens_host, self.lens = list(lens), torch.tensor(lens, dtype=torch.int32).cuda()
        shape = (*lead, self.pages, Hkv, page, d)
        code = torch.randint(0, 127, shape, generator=g, dtype=torch.uint8) | (torch.randint(0, 2, shape, generator=g, dtype=torch.uint8) << 7)
        code2 = code.flip(0)
        mk = lambda c: c.cuda().view(torch.float8_e4m3fn)  # noqa: E731
        self.kc, self.vc = mk(code), mk(code2.contiguous())
        if layout == "row_major":
            self.kc, self.vc = (t.transpose(-2, -3).contiguous().transpose(-2, -3) for t in (self.kc, self.vc))
        self.ks = torch.randint(117, 126, (*lead, self.pages, Hkv), generator=g, dtype=torch.uint8).cuda()
        self.vs = torch.randint(117, 126, (*lead, Hkv, self.pages), generator=g, dtype=torch.uint8).cuda().transpose(-1, -2)

    def host(self):
        raw = lambda t: t.contiguous().view(torch.uint8).cpu().numpy()  # noqa: E731
        return raw(self.kc), self.ks.cpu().numpy(), raw(self.vc), self.vs.contiguous().cpu().numpy()

    def scales(self):
        return dict(k_scale=self.ks, v_scale=self.vs)


def rows_of(seed, T, Hkv, d, dtype, odd=False):
    """New rows of magnitudes that differ between rows; heads 0 are small throughout."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, Hkv, d, generator=g) * torch.exp2(torch.randint(-6, 4, (T, 1, 1), generator=g).float())
    x[:, 0] *= 2.0 ** -6
    if odd and T:
        x[T // 2, Hkv - 1, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
        x[0, Hkv - 1] = 0
    return x.to(DT[dtype])


def equal(c, before, krows, vrows, starts, max_q=None):
    kc, ks, vc, vs = c.host()
    for codes, scales, c0, s0, rows, name in ((kc, ks, before[0], before[1], krows, "k"), (vc, vs, before[2], before[3], vrows, "v")):
        want, ws = R8.append(c0, s0, rows, c.table_host, c.lens_host, starts, max_q)
        assert np.array_equal(scales, ws), (name, np.argwhere(scales != ws)[:5], scales[scales != ws][:5], ws[scales != ws][:5])
        bad = ~R8.same(codes, want)
        assert not bad.any(), (name, int(bad.sum()), np.argwhere(bad)[:5], codes[bad][:5], want[bad][:5])


def positions(lens, starts):
    return np.concatenate([np.arange(n - (b - a), n) for n, a, b in zip(lens, starts, starts[1:])] + [np.zeros(0, int)])


# lens, news, Hkv, d, page
SHAPES = [
    ([1], [1], 1, 64, 16),
    ([33, 1, 70, 64, 65], [1, 1, 1, 1, 1], 4, 128, 16),   # single tokens: in a page, at a page's end, its first
    ([40, 300, 5], [5, 130, 5], 2, 128, 64),              # chunks; a whole prompt of 5
    ([65, 129], [33, 64], 3, 32, 24),                     # pages off every power of two
    ([9, 8, 17], [9, 0, 2], 2, 80, 8),                    # a sequence that brings nothing
    ([300], [299], 2, 64, 256),                           # a page of more rows than LDS holds angles for
    ([7, 500] + [3 + i for i in range(60)], [1, 400] + [1] * 60, 1, 64, 16),  # one prompt among single tokens
]
# dim of the rotated part (of d), interleaved, magnitude
ROTS = [(None, False), (1.0, False), (1.0, True), (0.5, False), (0.25, True)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_append8(shape, dtype):
    from nkilab import ops

    lens, news, Hkv, d, page = shape
    starts = [0] + list(np.cumsum(news))
    T = starts[-1]
    for i, (part, il) in enumerate(ROTS):
        c = Cache(i, lens, Hkv, d, page, layout=("page_major", "row_major")[i % 2])
        before = c.host()
        k, v = rows_of(i, T, Hkv, d, dtype, odd=i == 0), rows_of(i + 10, T, Hkv, d, dtype, odd=i == 1)
        r = None if part is None else ops.Rotary(max(2, int(d * part) // 2 * 2), 10000.0, interleaved=il, scaling="parts",
                                                 factor=4.0, original=64, magnitude=1.0 if i < 3 else 1.125)
        pos = positions(lens, starts)
        kw, H = {}, 2 * Hkv
        if r is not None:
            q = torch.randn(T, H, d, generator=torch.Generator().manual_seed(7)).to(DT[dtype]).cuda()
            q0 = q.clone()
            out = q if i == 2 else torch.full_like(q, float("nan"))
            kw = dict(q=q, q_out=out, rotary=r)
        ops.cache_append_into(k.cuda(), v.cuda(), c.kc, c.vc, c.table, c.lens, q_start=torch.tensor(starts, dtype=torch.int32).cuda(),
                              max_q=max(news), **kw, **c.scales())
        kd = k.double().numpy()
        equal(c, before, kd if r is None else R8.rotate(kd, pos, r), v.double().numpy(), starts)
        if r is not None:
            x = q0.double().cpu().numpy()
            want = R8.rotate(x, pos, r)
            err = np.abs(out.double().cpu().numpy() - want)
            assert (err <= R8.rotate_bound(x, want, r, torch.finfo(DT[dtype]))).all()


def test_append8_each_and_rope_base():
    """Without offsets; a rotary base in place of a table."""
    from nkilab import ops

    lens = [20, 33, 64]
    c = Cache(3, lens, 2, 64, 16)
    before = c.host()
    k, v = rows_of(1, 12, 2, 64, "bf16"), rows_of(2, 12, 2, 64, "bf16")
    ops.cache_append_into(k.cuda(), v.cuda(), c.kc, c.vc, c.table, c.lens, rope_base=500.0, **c.scales())
    starts = [0, 4, 8, 12]
    r = ops.Rotary(64, 500.0)
    equal(c, before, R8.rotate(k.double().numpy(), positions(lens, starts), r), v.double().numpy(), starts)


def test_append8_scale_follows_the_rows():
    """Row by row into one page, larger and smaller: the scale rises, never falls, and starts anew in the next page."""
    from nkilab import ops

    page, d = 8, 32
    c = Cache(0, [20], 1, d, page)
    amps = [1, 0.25, 40, 39, 1e-3, 900, 1e6, 0, 1e-7, 3e4, 0, 1e-30, 5, 2e38, 1e-38, 1, 0, 1e-45, 6e4, 1]
    g = torch.Generator().manual_seed(0)
    for j, a in enumerate(amps):
        x = (torch.randn(1, 1, d, generator=g) * a).clamp(-3e38, 3e38)
        c.lens_host, c.lens = [j + 1], torch.tensor([j + 1], dtype=torch.int32).cuda()
        before = c.host()
        ops.cache_append_into(x.cuda(), -x.cuda(), c.kc, c.vc, c.table, c.lens, **c.scales())
        equal(c, before, x.double().numpy(), -x.double().numpy(), [0, 1])


def test_append8_borders():
    """Values half way between codes, and largest magnitudes at and just past 448 times a power of two."""
    from nkilab import ops

    mids = np.concatenate((R8.MID, np.nextafter(R8.MID.astype(np.float32), np.float32(1e9)).astype(np.float64),
                           np.nextafter(R8.MID.astype(np.float32), np.float32(0)).astype(np.float64), R8.POS))
    for top in (448.0, np.nextafter(np.float32(448), np.float32(449)), 447.99, 224.0):
        x = np.zeros((4, 1, 128))
        x.reshape(-1)[:len(mids)] = mids
        x = np.minimum(x, top)
        x[0, 0, 0] = -top
        for e in (0, -20, 30):
            c = Cache(0, [4], 1, 128, 16)
            before = c.host()
            t = torch.from_numpy(x * 2.0 ** e).float()
            ops.cache_append_into(t.cuda(), -t.cuda(), c.kc, c.vc, c.table, c.lens, **c.scales())
            equal(c, before, t.double().numpy(), -t.double().numpy(), [0, 4])


def test_append8_tree_missing_pages_and_rest():
    """A node's position is its depth; rows with no page are not written, q is rotated all the same; rows past max_q,
    and of sequences that are shorter than they bring, are left."""
    from nkilab import ops

    g = torch.Generator().manual_seed(0)
    lens, news, Hkv, d, page = [40, 10, 5], [12, 6, 9], 2, 64, 8
    starts = [0, 12, 18, 27]
    c = Cache(1, lens, Hkv, d, page)
    c.table_host[0][4] = -1                 # rows 32 .. 39
    c.table_host[1][0] = c.pages + 3        # no such page
    c.table = torch.tensor(c.table_host, dtype=torch.int32).cuda()
    parents = [-1, 0, 0, 1, 3, 2, 5, 0, 7, 8, 8, 4, -1, 0, 1, 2, 3, 0] + [-1] + list(range(8))
    depth = []
    for s, e in zip(starts, starts[1:]):
        dd = []
        for p in parents[s:e]:
            dd.append(0 if p < 0 else dd[p] + 1)
        depth += dd
    qs = torch.tensor(starts, dtype=torch.int32).cuda()
    words = ops.tree_mask(torch.tensor(parents, dtype=torch.int32).cuda(), q_start=qs, max_q=12)
    r = ops.Rotary(64)
    k, v = rows_of(1, 27, Hkv, d, "bf16"), rows_of(2, 27, Hkv, d, "bf16")
    q = torch.randn(27, 4, d, generator=g).to(torch.bfloat16).cuda()
    out = torch.zeros_like(q)
    before = c.host()
    ops.cache_append_into(k.cuda(), v.cuda(), c.kc, c.vc, c.table, c.lens, q_start=qs, max_q=12, tree=words, q=q, q_out=out,
                          rotary=r, **c.scales())
    pos = np.concatenate([n - (e - s) + np.array(depth[s:e]) for n, s, e in zip(lens, starts, starts[1:])])
    equal(c, before, R8.rotate(k.double().numpy(), pos, r), v.double().numpy(), starts)
    want = R8.rotate(q.double().cpu().numpy(), pos, r)
    assert np.abs(out.double().cpu().numpy() - want).max() <= 2.0 ** -8 * np.abs(want).max()
    # no more than max_q rows of a sequence
    c = Cache(2, [30, 30], Hkv, d, page)
    before = c.host()
    q_start = torch.tensor([0, 9, 12], dtype=torch.int32).cuda()
    out = torch.full((12, 4, d), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.cache_append_into(k[:12].cuda(), v[:12].cuda(), c.kc, c.vc, c.table, c.lens, q_start=q_start, max_q=4, q=q[:12], q_out=out,
                          rotary=r, **c.scales())
    pos = np.concatenate((21 + np.arange(9), 27 + np.arange(3)))
    equal(c, before, R8.rotate(k[:12].double().numpy(), pos, r), v[:12].double().numpy(), [0, 9, 12], max_q=4)
    assert (out[4:9] == 7).all() and not (out[:4] == 7).all()


@pytest.mark.parametrize("dtype", DT)
def test_append_rotary_into_other_caches(dtype):
    """A table of frequencies over a cache that is not of 8 bits."""
    from nkilab import ops

    g = torch.Generator().manual_seed(4)
    for d, dim, il, page in ((64, 64, False, 16), (80, 40, True, 24), (128, 32, False, 64), (10, 6, True, 8)):
        lens, news, Hkv, H = [70, 33, 4], [40, 1, 4], 2, 6
        starts = [0, 40, 41, 45]
        pages = 20
        kc, vc = (torch.zeros(pages, Hkv, page, d, dtype=DT[dtype], device="cuda") for _ in range(2))
        perm = torch.randperm(pages, generator=g)
        cols = -(-70 // page)
        table = perm[:3 * cols].view(3, cols) if 3 * cols <= pages else torch.arange(3 * cols).view(3, cols) % pages
        if 3 * cols > pages:
            kc, vc = (torch.zeros(3 * cols, Hkv, page, d, dtype=DT[dtype], device="cuda") for _ in range(2))
            table = torch.randperm(3 * cols, generator=g).view(3, cols)
        qkv = torch.randn(45, (H + 2 * Hkv) * d, generator=g).to(DT[dtype]).cuda()
        q, k, v = (t.view(45, -1, d) for t in qkv.split([H * d, Hkv * d, Hkv * d], dim=1))
        r = ops.Rotary(dim, interleaved=il, scaling="bands", factor=4.0, original=32)
        x = qkv.double().cpu().numpy()
        ops.cache_append_into(k, v, kc, vc, table.int().cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                              q_start=torch.tensor(starts, dtype=torch.int32).cuda(), max_q=40, q=q, q_out=q, rotary=r)
        pos = positions(lens, starts)
        fi = torch.finfo(DT[dtype])
        xq, xk = x[:, :H * d].reshape(45, H, d), x[:, H * d:(H + Hkv) * d].reshape(45, Hkv, d)
        qr, kr = R8.rotate(xq, pos, r), R8.rotate(xk, pos, r)
        assert (np.abs(q.double().cpu().numpy() - qr) <= R8.rotate_bound(xq, qr, r, fi)).all()
        seq = np.repeat(np.arange(3), news)
        pg, off = table.numpy()[seq, pos // page], pos % page
        assert (np.abs(kc.double().cpu().numpy()[pg, :, off] - kr) <= R8.rotate_bound(xk, kr, r, fi)).all()
        assert np.array_equal(vc.double().cpu().numpy()[pg, :, off], x[:, (H + Hkv) * d:].reshape(45, Hkv, d))
        assert int((kc != 0).any(dim=(1, 3)).sum()) <= 45  # (no other row was written)


def test_unaligned_rows_and_other_stream():
    from nkilab import ops

    lens, starts = [20, 40], [0, 3, 13]
    base = torch.randn(13, 2 * 64 + 5, generator=torch.Generator().manual_seed(1)).to(torch.float16)
    for off in (1, 3):
        c = Cache(5, lens, 2, 64, 16)
        before = c.host()
        k = base.cuda()[:, off:off + 128].view(13, 2, 64)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            ops.cache_append_into(k, k, c.kc, c.vc, c.table, c.lens, q_start=torch.tensor(starts, dtype=torch.int32).cuda(), max_q=10,
                                  **c.scales())
        s.synchronize()
        rows = k.double().cpu().numpy()
        equal(c, before, rows, rows, starts)


def test_copy_pages_takes_scales():
    from nkilab import ops

    for lead in ((), (3,)):
        c = Cache(6, [100], 3, 64, 16, spare=6, lead=lead)
        before = c.host()
        pairs = [(0, 4), (1, 7), (2, 5), (0, 6)]
        ops.cache_copy_pages(c.kc, c.vc, pairs, **c.scales())
        after = c.host()
        ax = len(lead)
        for b, a in zip(before, after):
            want = b.copy()
            for s, t in pairs:
                want[(slice(None),) * ax + (t,)] = b[(slice(None),) * ax + (s,)]
            assert np.array_equal(a, want)


@pytest.mark.parametrize("page,d", [(4, 64), (8, 32), (16, 128), (24, 80), (64, 64)])
def test_accept8(page, d):
    from nkilab import ops

    rng = random.Random(page)
    layers, Hkv = 3, 3
    news = [12, 1, 40, 7, 30]
    lens = [n + rng.randrange(0, 90) for n in news]
    paths = [sorted(rng.sample(range(n), rng.randrange(0, min(n, 14) + 1))) for n in news]
    paths[2] = [0, 1, 2, 20, 21, 39]
    paths[4] = list(range(30))
    c = Cache(page, lens, Hkv, d, page, lead=(layers,))
    before = c.host()
    width = max(len(p) for p in paths)
    t = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32).cuda()
    starts = [0] + list(np.cumsum(news))
    out = ops.cache_accept(c.kc, c.vc, c.table, c.lens, t, q_start=torch.tensor(starts, dtype=torch.int32).cuda(), **c.scales())
    assert out.tolist() == [n - m + len(p) for n, m, p in zip(lens, news, paths)]
    after = c.host()
    for i in (0, 2):
        for layer in range(layers):
            want, ws = R8.accept(before[i][layer], before[i + 1][layer], c.table_host, lens, news, paths)
            assert np.array_equal(after[i + 1][layer], ws)
            bad = ~R8.same(after[i][layer], want)
            # rows behind a sequence's new length hold nothing
            for b, (n, m, p) in enumerate(zip(lens, news, paths)):
                for j in range(n - m + len(p), n):
                    bad[c.table_host[b][j // page], :, j % page] = False
            assert not bad.any(), (i, layer, np.argwhere(bad)[:5])


def test_graph_of_append8():
    """Captured, and replayed with other lengths, tables and rows."""
    from nkilab import ops

    c = Cache(8, [60, 61, 62], 2, 64, 16)
    k, v = (torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    r = ops.Rotary(64)
    q, out = torch.randn(3, 4, 64, device="cuda").bfloat16(), torch.empty(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    run = lambda: ops.cache_append_into(k, v, c.kc, c.vc, c.table, c.lens, q=q, q_out=out, rotary=r, **c.scales())  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for step, lens in enumerate(([17, 1, 40], [18, 2, 41], [33, 3, 42])):
        x = rows_of(step, 3, 2, 64, "bf16")
        k.copy_(x)
        v.copy_(-x)
        c.lens_host = lens
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        before = c.host()
        graph.replay()
        torch.cuda.synchronize()
        equal(c, before, R8.rotate(x.double().numpy(), np.array(lens) - 1, r), -x.double().numpy(), [0, 1, 2, 3])


def test_nothing_to_do():
    from nkilab import ops

    c = Cache(9, [5, 6], 2, 64, 16)
    before = c.host()
    e = torch.empty(0, 2, 64, device="cuda")
    ops.cache_append_into(e, e, c.kc, c.vc, c.table, c.lens, q_start=torch.zeros(3, dtype=torch.int32).cuda(), max_q=0, **c.scales())
    ops.cache_copy_pages(c.kc, c.vc, [], **c.scales())
    assert all(np.array_equal(a, b) for a, b in zip(before, c.host()))
