"""Products with 4-bit weights against their definition in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


class Weight:
    def __init__(self, N, K, group, zeros, sdt, seed):
        from nkilab import ops

        g = torch.Generator().manual_seed(seed)
        G = -(-K // group)
        self.codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
        self.scales = ((0.5 + torch.rand(N, G, generator=g)) / (4.6 * K ** 0.5)).to(DT[sdt])
        self.zeros = torch.randint(0, 16, (N, G), generator=g, dtype=torch.uint8) if zeros else None
        self.w = ops.pack_w4(self.codes.cuda(), self.scales.cuda(), None if not zeros else self.zeros.cuda(), group)
        spread = lambda t: np.repeat(t.double().numpy(), group, axis=1)[:, :K]  # noqa: E731
        self.q, self.s = self.codes.double().numpy(), spread(self.scales)
        self.z = spread(self.zeros) if zeros else np.full((N, K), 8.0)
        self.dense = (self.q - self.z) * self.s


def sums_bound(x, w):
    """How far the fp32 sums may be off: a group's sums run over (16 + q) x and
    (16 + z) x, each product exact, one rounding of 2^-24 of the magnitudes
    so far a term (2^-23 allows for the unit's own order and truncation), then three
    roundings where they are joined and scaled; and the groups' sums, at most K / 32
    roundings of the running output, which is below the scaled magnitudes."""
    K = x.shape[1]
    mags = np.abs(x) @ ((16 + w.q + 16 + w.z) * w.s).T
    return mags * 2.0 ** -23 * (min(K, 128) + 3 + K / 32)


def check(out, ref, bound, dtype):
    fi = torch.finfo(DT[dtype])
    err = np.abs(out.double().cpu().numpy() - ref)
    tol = bound + fi.eps / 2 * (np.abs(ref) + bound) + fi.tiny * fi.eps / 2
    assert (err <= tol).all(), (float((err / tol).max()), float(err.max()))
    # the bound above is the worst that signs could do; they are random here, and a sum of
    # n such errors is some sqrt(n) of them: a lost term, code or group is far outside this
    rms = np.sqrt((err ** 2).mean()) / np.sqrt((ref ** 2).mean())
    assert rms < max(fi.eps, 2e-6), rms


# M, N, K: single tokens, small and larger batches, sizes off every tile, fewer columns than a chunk
SHAPES = [(1, 16, 128), (1, 2048, 2048), (3, 100, 130), (16, 256, 512), (17, 33, 1000), (5, 1, 7), (40, 64, 96),
          (64, 48, 1024), (65, 130, 264), (200, 300, 136), (1, 5000, 4224), (129, 257, 1990)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_w4(M, N, K, dtype):
    from nkilab import ops

    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g).to(DT[dtype])
    xd = x.double().numpy()
    for i, group in enumerate((32, 64, 128, 256)):
        w = Weight(N, K, group, zeros=i % 2 == 0, sdt=dtype if i < 2 else "fp32", seed=i)
        ref, bound = xd @ w.dense.T, sums_bound(xd, w)
        y = torch.full((M, N), float("nan"), dtype=DT[dtype], device="cuda")
        assert ops.linear_w4_into(x.cuda(), w.w, y) is y
        check(y, ref, bound, dtype)
        # into fp32 rows of a wider tensor, onto the residual that is there
        wide = torch.randn(M, N + 3, generator=g).cuda()
        keep, res = wide.clone(), wide[:, 1:N + 1].double().cpu().numpy()
        ops.linear_w4_into(x.cuda(), w.w, wide[:, 1:N + 1], residual=wide[:, 1:N + 1])
        check(wide[:, 1:N + 1], ref + res, bound + 2.0 ** -24 * np.abs(res), "fp32")
        assert torch.equal(wide[:, 0], keep[:, 0]) and torch.equal(wide[:, N + 1:], keep[:, N + 1:])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,N,K", [(1, 64, 256), (2, 40, 200), (33, 704, 520), (70, 17, 128), (150, 96, 384)])
def test_swiglu_w4(M, N, K, dtype):
    from nkilab import ops

    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).to(DT[dtype])
    xd = x.double().numpy()
    for group in (32, 128):
        a, b = Weight(N, K, group, True, dtype, 1), Weight(N, K, group, True, dtype, 2)
        gate, up = xd @ a.dense.T, xd @ b.dense.T
        silu = gate / (1 + np.exp(-gate))
        # silu's slope is at most 1.1; its own exponential, reciprocal and products: 2^-20 of it
        bound = 1.1 * sums_bound(xd, a) * (np.abs(up) + 1) + sums_bound(xd, b) * (np.abs(silu) + 1) + 2.0 ** -20 * np.abs(silu * up)
        y = torch.empty(M, N, dtype=DT[dtype], device="cuda")
        ops.linear_w4_swiglu_into(x.cuda(), ops.pair_w4(a.w, b.w), y)
        check(y, silu * up, bound, dtype)


def test_swiglu_of_large_gates():
    """Gates so far from zero that the exponential overflows or vanishes."""
    from nkilab import ops

    codes = torch.tensor([[15] * 128, [0] * 128], dtype=torch.uint8).cuda()
    w = ops.pack_w4(codes, torch.ones(2, 1).cuda())
    x = torch.full((1, 128), 10.0).cuda()
    y = ops.linear_w4_swiglu_into(x, ops.pair_w4(w, w), torch.empty(1, 2, device="cuda"))
    assert y.cpu().tolist() == [[8960.0 ** 2, 0.0]]


def test_views_and_alignment():
    """Rows of x at odd addresses, a transposed x, and outputs that no vector store fits."""
    from nkilab import ops

    g = torch.Generator().manual_seed(0)
    for dtype in DT:
        w = Weight(50, 203, 64, True, dtype, 5)
        base = torch.randn(9, 300, generator=g).to(DT[dtype]).cuda()
        for x in (base[:, 1:204], base[:, 3:206], torch.randn(203, 9, generator=g).to(DT[dtype]).cuda().t(), base[2:3, 7:210]):
            xd = x.double().cpu().numpy()
            y = torch.zeros(x.shape[0], 53, dtype=DT[dtype], device="cuda")
            ops.linear_w4_into(x, w.w, y[:, 3:])
            check(y[:, 3:], xd @ w.dense.T, sums_bound(xd, w), dtype)
            assert not y[:, :3].any()


def test_rows_do_not_meet():
    """An infinity or NaN in one row of x stays there."""
    from nkilab import ops

    for M in (5, 70):
        w = Weight(40, 256, 128, False, "bf16", 5)
        x = torch.randn(M, 256).to(torch.bfloat16).cuda()
        want = ops.linear_w4(x, w.w)
        x[1, 3], x[3, 200] = float("inf"), float("nan")
        y = ops.linear_w4(x, w.w)
        rest = [i for i in range(M) if i not in (1, 3)]
        assert torch.equal(y[rest], want[rest]) and y[[1, 3]].isnan().all()


def test_quantize_and_unpack():
    from nkilab import ops

    g = torch.Generator().manual_seed(1)
    w = torch.randn(70, 300, generator=g).cuda()
    w[3] = 0
    for zeros in (False, True):
        for group in (32, 128):
            q = ops.quantize_w4(w, group, zeros=zeros)
            d = ops.unpack_w4(q)
            # a value is off by at most half a step, which is the group's largest / 7, or range / 15
            # (with zeros rounded to a code: a whole one at the ends)
            x = torch.nn.functional.pad(w, (0, -300 % group)).view(70, -1, group)
            step = (x.amax(2) - x.amin(2)) / 15 if zeros else x.abs().amax(2) / 7
            lim = step.clamp(min=0).repeat_interleave(group, 1)[:, :300] * (1.001 if zeros else 0.5005) + 1e-12
            assert ((d - w).abs() <= lim).all() and not d[3].any()
            x1 = torch.randn(1, 300, generator=g).cuda()
            y = ops.linear_w4(x1, q).double()
            assert ((y - x1.double() @ d.double().t()).abs() < 1e-3).all()


def test_kinds_empty_streams_graphs():
    from nkilab import ops

    w = Weight(64, 256, 64, True, "fp32", 2)
    x = torch.randn(6, 256)
    y = ops.linear_w4(x.numpy(), w.w)
    assert isinstance(y, np.ndarray)
    assert ops.linear_w4(x[:0].cuda(), w.w).shape == (0, 64)
    xg, out = x.cuda(), torch.empty(6, 64, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.linear_w4_into(xg, w.w, out)
    s.synchronize()
    assert np.array_equal(out.cpu().numpy(), y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_w4_into(xg, w.w, out)
    for k in range(3):
        xg.copy_(torch.randn(6, 256))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.linear_w4(xg, w.w))


# Enough of them for narrow tiles in two groups (one block of rows, and two; one, two and
# three chunks) and in one group, for those half as wide, and for wide ones with more than
# four blocks of rows (M, N, K with edges inside every tile)
TILES = [(40, 4200, 72), (40, 4200, 136), (70, 2117, 264), (70, 8300, 136), (200, 8300, 264), (530, 6603, 200)]


@pytest.mark.parametrize("dtype,sdt", [(d, s) for d in DT for s in dict.fromkeys((d, "fp32"))])
@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles_w4(M, N, K, dtype, sdt):
    from nkilab import ops

    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g).to(DT[dtype])
    xd = x.double().numpy()
    for i, group in enumerate((32, 64, 128, 256)):
        w = Weight(N, K, group, zeros=i % 2 == 1, sdt=sdt, seed=i)
        y = torch.full((M + 1, N), 7.0, dtype=DT[dtype], device="cuda")
        ops.linear_w4_into(x.cuda(), w.w, y[:M])
        check(y[:M], xd @ w.dense.T, sums_bound(xd, w), dtype)
        assert (y[M] == 7).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,N,K", [(70, 1060, 264), (70, 4200, 264), (200, 4200, 136), (330, 3300, 136)])
def test_swiglu_tiles_w4(M, N, K, dtype):
    from nkilab import ops

    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).to(DT[dtype])
    xd = x.double().numpy()
    for group in (64, 128):
        a, b = Weight(N, K, group, True, dtype, 1), Weight(N, K, group, True, dtype, 2)
        gate, up = xd @ a.dense.T, xd @ b.dense.T
        silu = gate / (1 + np.exp(-gate))
        bound = 1.1 * sums_bound(xd, a) * (np.abs(up) + 1) + sums_bound(xd, b) * (np.abs(silu) + 1) + 2.0 ** -20 * np.abs(silu * up)
        y = ops.linear_w4_swiglu_into(x.cuda(), ops.pair_w4(a.w, b.w), torch.empty(M, N, dtype=DT[dtype], device="cuda"))
        check(y, silu * up, bound, dtype)


def test_infinities_in_tiles():
    """As test_rows_do_not_meet, where 16 rows of a tile are multiplied at once."""
    from nkilab import ops

    w = Weight(4200, 264, 128, True, "bf16", 5)
    x = torch.randn(70, 264, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    want = ops.linear_w4(x, w.w)
    x[1, 3], x[65, 263] = float("inf"), float("nan")
    y = ops.linear_w4(x, w.w)
    rest = [i for i in range(70) if i not in (1, 65)]
    assert torch.equal(y[rest], want[rest]) and y[[1, 65]].isnan().all()


def test_two_products_at_once():
    """Two streams, one weight: nothing is shared between calls but what they read."""
    from nkilab import ops

    g = torch.Generator().manual_seed(3)
    w = Weight(2117, 264, 64, True, "fp16", 2)
    xs = [torch.randn(m, 264, generator=g).to(torch.float16).cuda() for m in (1, 70)]
    want = [ops.linear_w4(x, w.w) for x in xs]
    outs = [torch.empty_like(y) for y in want]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, x, y in zip(streams, xs, outs):
            with torch.cuda.stream(s):
                ops.linear_w4_into(x, w.w, y)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
