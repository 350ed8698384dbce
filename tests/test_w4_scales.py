"""Scales that quantize_w4 chooses where their type has few numbers left, with no GPU."""
import pytest
import torch

# type, exponents of the group's largest magnitude: from normal scales to the smallest subnormal one
TYPES = [(torch.float16, range(-27, -8)), (torch.bfloat16, range(-136, -120)), (torch.float32, range(-146, -120))]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype,exponents", TYPES)
def test_quantize_small_values(dtype, exponents, zeros):
    """What is unpacked is within half a step of the scale that is stored (with zeros, whose codes are
    rounded too, a whole one), also where scales are subnormal numbers of their type."""
    from nkilab import ops

    g = torch.Generator().manual_seed(0)
    for e in exponents:
        w = torch.randn(16, 256, generator=g).clamp(-4, 4).double() * 2.0 ** e
        w[1] = w[1].abs()
        w[2] = -w[2].abs()
        w = w.float()  # (values that fp32 holds, some of them subnormal)
        q = ops.quantize_w4(w, 64, zeros=zeros, scale_dtype=dtype)
        step = q.scales.transpose(1, 2).reshape(16, -1).double().repeat_interleave(64, 1)
        assert q.scales.dtype is dtype
        err = (ops.unpack_w4(q).double() - w.double()).abs()
        # quotients are rounded to 24 bits before they are rounded to codes; a normal scale is
        # itself rounded, by half a step of its type, which the largest codes multiply by up to 15
        slack = 2.0 ** -20 + (0 if zeros else 8 * torch.finfo(dtype).eps / 2)
        assert (err <= step * ((1.0 if zeros else 0.5) + slack) + 2.0 ** -150).all(), (e, float((err / step.clamp(min=1e-300)).max()))
        # and the step is no larger than it has to be: the next smaller number of the type at most
        x = w.view(16, 4, 64).double()
        need = (x.amax(2).clamp(min=0) - x.amin(2).clamp(max=0)) / 15 if zeros else torch.maximum(x.amax(2) / 7, x.amin(2) / -8)
        least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the subnormal numbers' distance
        assert (q.scales.transpose(1, 2).reshape(16, 4).double() <= need * (1 + torch.finfo(dtype).eps) + least).all()


@pytest.mark.parametrize("std", [1e-3, 1e-4, 1e-5])
def test_quantize_small_fp16_weight(std):
    """A weight of fp16 keeps its scales' type, and as much of its values as one of fp32 does."""
    from nkilab import ops

    w = (torch.randn(32, 256, generator=torch.Generator().manual_seed(1)) * std).half()
    rel = lambda q: float((ops.unpack_w4(q) - w.float()).norm() / w.float().norm())  # noqa: E731
    wide = rel(ops.quantize_w4(w, 64, scale_dtype=torch.float32))
    # (a group's largest value is some 2.5 std: at 1e-5 its scale is 60 of the smallest subnormal number,
    # which rounded up is a step larger by a sixtieth at most; nearest codes' errors are a step's 0.29)
    assert rel(ops.quantize_w4(w, 64)) <= 1.05 * wide < 0.2


def test_weights_of_any_strides():
    """Codes, scales and zeros that are transposed or shared between rows, a transposed weight."""
    from nkilab import ops

    g = torch.Generator().manual_seed(4)
    codes = torch.randint(0, 16, (128, 48), generator=g, dtype=torch.uint8)
    scales, zeros = torch.rand(1, 2, generator=g).expand(48, 2), torch.full((1, 1), 3, dtype=torch.uint8).expand(48, 2)
    w = ops.pack_w4(codes.t(), scales, zeros, 64)
    assert torch.equal(ops.unpack_w4(w), (codes.t().float() - 3) * scales.repeat_interleave(64, 1))
    m = torch.randn(128, 48, generator=g)
    a, b = ops.quantize_w4(m.t(), 64), ops.quantize_w4(m.t().contiguous(), 64)
    assert torch.equal(a.packed, b.packed) and torch.equal(a.scales, b.scales)
