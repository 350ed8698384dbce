"""Products with 4-bit weights of activations with a mean, and of codes that lie close to their zeros:
what is left of such sums is far below the magnitudes of codes and activations."""
import numpy as np
import pytest
import torch

from test_gpu_w4 import DT, sums_bound

pytestmark = pytest.mark.gpu

# every kernel's rows and tiles, and a longer sum
SIZES = [(1, 100, 4096), (5, 40, 130), (20, 64, 264), (40, 96, 2048), (70, 2117, 264), (70, 4200, 264), (200, 8300, 264)]


class Close:
    """Codes within one of their zeros."""

    def __init__(self, N, K, group, zeros, sdt, seed, spread=1):
        from nkilab import ops

        g = torch.Generator().manual_seed(seed)
        G = -(-K // group)
        zero = torch.randint(1, 15, (N, G), generator=g) if zeros else torch.full((N, G), 8)
        wide = zero.repeat_interleave(group, 1)[:, :K]
        codes = (wide + torch.randint(-spread, spread + 1, (N, K), generator=g)).to(torch.uint8)
        scales = ((0.5 + torch.rand(N, G, generator=g)) / K ** 0.5).to(DT[sdt])
        self.w = ops.pack_w4(codes.cuda(), scales.cuda(), zero.to(torch.uint8).cuda() if zeros else None, group)
        self.q, self.z = codes.double().numpy(), wide.double().numpy()
        self.s = np.repeat(scales.double().numpy(), group, axis=1)[:, :K]
        self.dense = (self.q - self.z) * self.s


def activations(M, K, mean, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(M, K, generator=g) + mean).to(DT[dtype])


@pytest.mark.parametrize("mean", [1.0, 10.0])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_fp32_sums(M, N, K, mean):
    """fp32 activations: the products (q - z) x are summed, whatever x's mean.

    A running sum has K products and K / 32 sums of groups; a term is three parts of x, each product
    exact.  Each of some 3 K roundings is at most 2^-23 (truncation) of the sum so far, which is of the
    size of the result or below it (signs are random), and their signs are random: together sqrt(3 K)
    of them, 2^-23 sqrt(3 K) / sqrt(3) of the result."""
    from nkilab import ops

    x = activations(M, K, mean, "fp32", M)
    xd = x.double().numpy()
    for i, group in enumerate((32, 64, 128, 256)):
        w = Close(N, K, group, i % 2 == 0, "fp32", i)
        y = ops.linear_w4_into(x.cuda(), w.w, torch.empty(M, N, device="cuda")).double().cpu().numpy()
        ref = xd @ w.dense.T
        rms = np.sqrt(((y - ref) ** 2).mean() / (ref ** 2).mean())
        assert rms <= 2.0 ** -23 * K ** 0.5, rms


@pytest.mark.parametrize("M,N,K", SIZES)
def test_fp32_codes_at_zero(M, N, K):
    """Codes that are their zeros: exactly 0, with any scale."""
    from nkilab import ops

    x = activations(M, K, 10.0, "fp32", M)
    for group, zeros in ((32, True), (64, False), (128, True), (256, False)):
        w = Close(N, K, group, zeros, "fp32", 1, spread=0)
        assert not ops.linear_w4_into(x.cuda(), w.w, torch.full((M, N), 7.0, device="cuda")).any()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_fp32_large_activations(M, N, K):
    """Sums that fp32 holds, of activations whose products with 16 + q it would not."""
    from nkilab import ops

    x = activations(M, K, 0.0, "fp32", M).clamp(-4, 4) * 2.0 ** 122
    for group, zeros in ((32, True), (128, False)):
        w = Close(N, K, group, zeros, "fp32", 1)
        w.w.scales[:] *= 2.0 ** -10
        y = ops.linear_w4_into(x.cuda(), w.w, torch.empty(M, N, device="cuda")).double().cpu().numpy()
        ref = x.double().numpy() @ (w.dense * 2.0 ** -10).T
        assert np.sqrt(((y - ref) ** 2).mean() / (ref ** 2).mean()) <= 2.0 ** -23 * K ** 0.5


@pytest.mark.parametrize("mean", [1.0, 10.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_16_bit_sums(M, N, K, dtype, mean):
    """16-bit activations: sums are of (16 + q) x, and as exact as their magnitudes allow."""
    from nkilab import ops

    x = activations(M, K, mean, dtype, M)
    xd = x.double().numpy()
    for i, group in enumerate((32, 64, 128, 256)):
        w = Close(N, K, group, i % 2 == 0, dtype, i)
        y = ops.linear_w4_into(x.cuda(), w.w, torch.empty(M, N, device="cuda")).double().cpu().numpy()
        ref, bound = xd @ w.dense.T, sums_bound(xd, w)
        assert (np.abs(y - ref) <= bound + 2.0 ** -24 * np.abs(ref)).all()
        # (random signs: the square root of the bound's K / 32 + 128 roundings a term)
        n = min(K, 128) + 3 + K / 32
        assert np.sqrt(((y - ref) ** 2).mean()) <= np.sqrt((bound ** 2).mean() / n)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,N,K", [(5, 40, 130), (20, 64, 264), (70, 2117, 264), (200, 8300, 264)])
def test_rows_with_infinities(M, N, K, dtype):
    """An infinity or NaN makes its row NaN, also where its codes are their zeros, and no other."""
    from nkilab import ops

    x = activations(M, K, 0.0, dtype, M).cuda()
    for zeros, spread in ((True, 1), (False, 0)):
        w = Close(N, K, 64, zeros, "fp32", 2, spread=spread)
        want = ops.linear_w4(x, w.w)
        odd = x.clone()
        odd[1, K - 1], odd[2, 3], odd[4, 64] = float("-inf"), float("nan"), float("inf")
        if dtype == "fp32":  # a NaN whose upper half is an infinity's
            odd.view(torch.int32)[3, 5] = 0x7f800001
        y = ops.linear_w4(odd, w.w)
        bad = [1, 2, 4] + ([3] if dtype == "fp32" else [])
        rest = [i for i in range(M) if i not in bad]
        assert y[bad].isnan().all() and torch.equal(y[rest], want[rest])
