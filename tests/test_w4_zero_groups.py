"""Groups of zeros in quantize_w4, with no GPU."""
import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
def test_scales_of_zero_groups(zeros, dtype):
    """A group without a value that is not 0 has scale 0, so that its products are exactly 0; the
    groups beside it have theirs."""
    from nkilab import ops

    w = torch.randn(20, 300, generator=torch.Generator().manual_seed(2)).to(dtype)
    w[3] = 0
    w[5, 64:128] = 0
    w[6, 256:] = 0
    q = ops.quantize_w4(w, 64, zeros=zeros)
    s = q.scales.transpose(1, 2).reshape(32, -1)[:20, :5]
    none = torch.zeros(20, 5, dtype=torch.bool)
    none[3], none[5, 1], none[6, 4] = True, True, True
    assert torch.equal(s == 0, none)
    d = ops.unpack_w4(q)
    assert not d[3].any() and not d[5, 64:128].any() and not d[6, 256:].any() and d[5, :64].any()


def test_least_values_are_not_zeros():
    """The smallest number there is has a scale, the smallest too."""
    from nkilab import ops

    w = torch.zeros(2, 32)
    w[0, 3], w[1, 5] = 2.0 ** -149, -3 * 2.0 ** -149
    for zeros in (False, True):
        q = ops.quantize_w4(w, 32, zeros=zeros)
        assert torch.equal(ops.unpack_w4(q), w) and (q.scales[0, 0, :2] == 2.0 ** -149).all()
