"""Rotary bases that 32 bits do not hold, on the GPU."""
import numpy as np
import pytest
import torch

import paged_reference as R
from test_gpu_paged import DT, rope_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("base", [82684.62, 1234567.891, 10000.0])
def test_rotary_bases_are_taken_in_64_bits(dtype, base):
    """Far positions: a base rounded to 32 bits is off by up to 1e-4 radians there."""
    from nkilab import ops

    d, page, far = 128, 64, 131072 + 5
    pages = -(-far // page)
    kc = torch.zeros(3, 1, page, d, dtype=DT[dtype], device="cuda")
    vc = torch.zeros_like(kc)
    table = torch.full((1, pages), -1, dtype=torch.int32)
    table[0, -2:] = torch.tensor([2, 1])
    g = torch.Generator().manual_seed(52)
    k = torch.randn(9, 1, d, generator=g).to(DT[dtype]).cuda()
    q = torch.randn(9, 2, d, generator=g).to(DT[dtype]).cuda()
    q_out = torch.empty_like(q)
    lens = torch.tensor([far], dtype=torch.int32).cuda()
    ops.cache_append_into(k, k, kc, vc, table.cuda(), lens, q=q, q_out=q_out, rope_base=base)
    x, xmax = q.double().cpu().numpy(), float(q.float().abs().max())
    want = np.stack([R.rope(x[i], far - 9 + i, base) for i in range(9)])
    rope_close(q_out, want, dtype, xmax)
    xk = k.double().cpu().numpy()
    want = np.stack([R.rope(xk[i], far - 9 + i, base) for i in range(9)])
    rows = [(2, j) for j in range(60, 64)] + [(1, j) for j in range(5)]  # positions 131068 .. 131076
    rope_close(torch.stack([kc[p, :, j] for p, j in rows]), want, dtype, float(k.float().abs().max()))
