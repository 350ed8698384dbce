"""Offsets of new rows that a caller should not make: sequences that overlap."""
import pytest
import torch

from test_gpu_paged import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("times", [2, 51, 130])
@pytest.mark.parametrize("n,length", [(512, 2080), (512, 513), (20, 3000)])
def test_sequences_that_name_the_same_rows(n, length, times, dtype):
    """More row tiles than the packed rows have, all of them worked on: every
    second sequence names all the rows (the others none), over the same pages."""
    from nkilab import ops

    b = Batch(60, [length], [n], 1, 1, 64, 16, dtype)
    batch = 2 * times - 1
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens = b.table.expand(batch, -1).contiguous(), torch.full((batch,), length, **i32)
    q_start = torch.tensor([0, n] * times, **i32)
    for window in (None, 300):
        b.check(ops.paged_attention(b.q, b.kc, b.vc, table, lens, q_start=q_start, max_q=n, window=window), window=window)
