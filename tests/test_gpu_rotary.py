"""Rotary positions with a table of frequencies, against their definition in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def formula(x, pos, r, grad=False):
    """x [H, S, d] in 64 bits, one pair at a time."""
    y = x.copy()
    for i, f in enumerate(r.frequencies):
        a, b = (2 * i, 2 * i + 1) if r.interleaved else (i, i + r.dim // 2)
        t = np.asarray(pos, np.float64) * f
        c, s = r.gain * np.cos(t), r.gain * np.sin(t) * (-1 if grad else 1)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def bound(x, y, r, dtype):
    """Sine and cosine are rounded to fp32, so are two products and their sum
    (2^-24 of at most gain (|x1| + |x2|) each), and the output to its type by half a
    step (of a value that is off by the former; below the type's normal numbers half
    a step of the smallest of those).  The 64-bit angles' own errors are within
    2^-53 * 2^20 positions."""
    half = r.dim // 2
    pair = np.zeros(x.shape)
    a, b = (slice(0, r.dim, 2), slice(1, r.dim, 2)) if r.interleaved else (slice(0, half), slice(half, r.dim))
    pair[..., a] = pair[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    inner = (3 * 2.0 ** -24 + 2.0 ** -30) * abs(r.gain) * pair
    fi = torch.finfo(DT[dtype])
    return inner + fi.eps / 2 * (np.abs(y) + inner) + fi.tiny * fi.eps / 2


def check(out, x, pos, r, dtype, grad=False):
    x = x.double().cpu().numpy()
    want = formula(x, pos, r, grad)
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= bound(x, want, r, dtype)).all(), (err.max(), r)


def make(H, S, d, dtype, seed=0, layout="hsd"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(S, H, d, generator=g).to(DT[dtype]).cuda()
    return x.transpose(0, 1) if layout == "shd" else x.transpose(0, 1).contiguous()


SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
            dict(scaling="parts", factor=16.0, original=4096), dict(scaling="bands", factor=8.0, original=8192),
            dict(scaling="parts", factor=2.0, original=100, low_turns=0.5, high_turns=3.0, magnitude=0.7)]

# H, S, d, dim: vector and scalar widths, part of the head, one row, one pair, odd heads
SHAPES = [(1, 1, 64, 64), (40, 64, 128, 128), (5, 37, 128, 64), (3, 513, 80, 40), (2, 70, 256, 256), (7, 33, 96, 2),
          (1, 3, 10, 6), (4, 100, 66, 34), (300, 2, 64, 32)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,S,d,dim", SHAPES)
def test_rotary_matches_formula(H, S, d, dim, dtype, interleaved):
    from nkilab import ops

    for k, sc in enumerate(SCALINGS):
        r = ops.Rotary(dim, 10000.0 if k % 2 else 500000.0, interleaved=interleaved, **sc)
        x = make(H, S, d, dtype, seed=k, layout=("hsd", "shd")[k % 2])
        g = torch.Generator().manual_seed(k)
        pos = torch.randint(0, 1 << 20, (S,), generator=g, dtype=torch.int32 if k % 3 else torch.int64)
        grad = k in (2, 4)
        y = torch.full_like(x, float("nan"))
        assert ops.rotary_into(x, y, r, positions=pos.cuda(), grad=grad) is y
        check(y, x, pos.numpy(), r, dtype, grad)
        # from one position on; in place
        z = x.clone()
        ops.rotary_into(z, z, r, pos0=5 + k, grad=grad)
        check(z, x, 5 + k + np.arange(S), r, dtype, grad)


def test_far_and_negative_positions():
    from nkilab import ops

    r = ops.Rotary(64)
    x = make(2, 6, 64, "fp32")
    pos = [0, -1, -100000, (1 << 30) + 1, (1 << 31) - 1, -(1 << 31)]
    y = ops.rotary(x, r, positions=torch.tensor(pos))
    assert y.is_cuda
    # The formula's angle, position * frequency in 64 bits, is the kernel's own product: what is
    # left is its reduction by multiples of pi / 2 (at most 2^31 of them, their product exact).
    check(y, x, np.array(pos), r, "fp32")


def test_strided_views_and_rest_of_a_projection():
    """q and k as columns of a projection's rows, rotated in place: the v columns stay."""
    from nkilab import ops

    g = torch.Generator().manual_seed(3)
    S, H, Hkv, d = 45, 6, 2, 64
    qkv = torch.randn(S, (H + 2 * Hkv) * d, generator=g).to(torch.bfloat16).cuda()
    before = qkv.clone()
    r = ops.Rotary(32, interleaved=True)
    qk = qkv[:, :(H + Hkv) * d].view(S, H + Hkv, d).transpose(0, 1)
    ops.rotary_into(qk, qk, r)
    assert torch.equal(qkv[:, (H + Hkv) * d:], before[:, (H + Hkv) * d:])
    check(qk, before[:, :(H + Hkv) * d].view(S, H + Hkv, d).transpose(0, 1), np.arange(S), r, "bf16")
    # rows that are not on 16 bytes
    odd = torch.randn(4, 9, 67, generator=g).cuda()
    x = odd[:, :, 1:65]
    y = torch.empty(4, 9, 65, device="cuda")[:, :, 1:]
    ops.rotary_into(x, y, r)
    check(y, x, np.arange(9), r, "fp32")


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_by_differences(interleaved):
    """The map is linear: (f(x + v) - f(x - v)) / 2 is its value at v, and g . f(v) = grad(g) . v."""
    from nkilab import ops

    r = ops.Rotary(48, scaling="parts", factor=8.0, original=512, interleaved=interleaved)
    x, v, g = (make(3, 50, 64, "fp32", seed=s) for s in (1, 2, 3))
    f = lambda t: ops.rotary(t, r, pos0=1000).double()  # noqa: E731
    left = ((f(x + v) - f(x - v)) / 2 * g.double()).sum().item()
    right = (ops.rotary(g, r, pos0=1000, grad=True).double() * v.double()).sum().item()
    # each of 2 * 9600 terms is off by a few 2^-24 of values of up to 1.3 * 2 * 5 * 5; their sum by less than
    # the sum of magnitudes, which is below 9600 * 65 * 8 * 2^-24
    assert abs(left - right) < 9600 * 65 * 8 * 2.0 ** -24
    assert abs(left) > 1.0


def test_kinds_streams_and_graphs():
    from nkilab import ops

    r = ops.Rotary(64, scaling="linear", factor=2.0)
    x = make(4, 20, 64, "fp32")
    want = ops.rotary(x, r, pos0=3)
    a = ops.rotary(x.cpu().numpy(), r, pos0=3)
    assert isinstance(a, np.ndarray) and np.array_equal(a, want.cpu().numpy())
    assert torch.equal(ops.rotary(x.cpu(), r, positions=3 + torch.arange(20)), want.cpu())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y, pos = torch.empty_like(x), torch.arange(20, dtype=torch.int32, device="cuda")
    with torch.cuda.stream(s):
        ops.rotary_into(x, y, r, positions=pos)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary_into(x, y, r, positions=pos)
    for shift in (0, 7, 900000):
        pos.copy_(torch.arange(20, dtype=torch.int32) + shift)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.rotary(x, r, pos0=shift))


def test_empty():
    from nkilab import ops

    for shape in ((0, 4, 64), (3, 0, 64)):
        x = torch.empty(shape, device="cuda")
        assert ops.rotary(x, ops.Rotary(64)).shape == shape
