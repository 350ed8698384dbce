"""Products with 4-bit weights where sums cancel: zero groups, subnormal scales, activations with a mean."""
import numpy as np
import pytest
import torch

from test_gpu_w4 import DT, Weight, check, sums_bound

pytestmark = pytest.mark.gpu

# rows of one and of two fragments, and enough rows and tiles for each kind of tile kernel
SIZES = [(1, 70, 512), (20, 64, 264), (70, 2117, 264), (200, 8300, 264)]


class Quantized:
    """quantize_w4's weight as Weight has one, for sums_bound."""

    def __init__(self, w, K):
        spread = lambda t: np.repeat(t.transpose(1, 2).reshape(-1, t.shape[1]).double().cpu().numpy(),  # noqa: E731
                                     w.group, axis=1)[:w.n, :K]
        self.s = spread(w.scales)
        self.z = spread(w.zeros) if w.zeros is not None else np.full((w.n, K), 8.0)
        from nkilab import ops

        self.dense = ops.unpack_w4(w).double().cpu().numpy()
        with np.errstate(divide="ignore", invalid="ignore"):
            self.q = np.where(self.s > 0, np.rint(self.dense / self.s) + self.z, self.z)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_zero_rows_and_groups(M, N, K, dtype):
    """Rows of zeros give exactly 0, whatever x's mean; rows of some zero groups what the others do."""
    from nkilab import ops

    g = torch.Generator().manual_seed(N)
    w = torch.randn(N, K, generator=g) / K ** 0.5
    w[3] = 0
    w[5, 64:256] = 0
    x = (torch.randn(M, K, generator=g) + 10).to(DT[dtype])
    for zeros in (False, True):
        for group in (32, 64, 128):
            q = ops.quantize_w4(w.cuda(), group, zeros=zeros, scale_dtype=torch.float32)
            y = ops.linear_w4_into(x.cuda(), q, torch.empty(M, N, device="cuda"))
            assert not y[:, 3].any()
            ref, xd = Quantized(q, K), x.double().numpy()
            exact = xd @ ref.dense.T
            assert (np.abs(y.double().cpu().numpy() - exact) <= sums_bound(xd, ref) + 2.0 ** -24 * np.abs(exact)).all()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_subnormal_scales(M, N, K):
    """An fp16 weight of small values, whose scales are subnormal."""
    from nkilab import ops

    g = torch.Generator().manual_seed(N)
    w = (torch.randn(N, K, generator=g) * 1e-5).half()
    x = (torch.randn(M, K, generator=g) * 1000).half()
    for zeros in (False, True):
        q = ops.quantize_w4(w.cuda(), 64, zeros=zeros)
        assert 0 < float(q.scales.max()) < torch.finfo(torch.float16).smallest_normal
        ref = Quantized(q, K)
        step = ref.s * (1 if zeros else 0.5)
        assert (np.abs(ref.dense - w.double().numpy()) <= step * (1 + 2.0 ** -19)).all()
        y = ops.linear_w4_into(x.cuda(), q, torch.empty(M, N, dtype=torch.float16, device="cuda"))
        check(y, x.double().numpy() @ ref.dense.T, sums_bound(x.double().numpy(), ref), "fp16")
