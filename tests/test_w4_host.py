"""Packed 4-bit weights on the CPU, and what their entry points refuse, with no GPU."""
import pytest
import torch

P = 1 << 20  # (an aligned address, refused before it is used)


def test_packed_layout():
    """Every code is where the C header says it is."""
    from nkilab import ops

    g = torch.Generator().manual_seed(0)
    N, K, group = 37, 300, 64
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    scales = torch.rand(N, 5, generator=g) + 0.5
    zeros = torch.randint(0, 16, (N, 5), generator=g, dtype=torch.uint8)
    w = ops.pack_w4(codes, scales, zeros, group)
    raw = w.packed.contiguous().numpy().tobytes()
    assert len(raw) == 3 * 3 * 1024 and w.scales.shape == (3, 6, 16) and w.zeros.shape == (3, 6, 16)
    for n, k in ((0, 0), (1, 1), (15, 127), (16, 128), (36, 299), (20, 250), (7, 66)):
        t, c, r, kk = n // 16, k // 128, n % 16, k % 128
        s, lane, j = kk // 32, 16 * (kk % 32 // 8) + r, kk % 8
        at = (t * 3 + c) * 1024 + lane * 16 + 4 * s
        word = int.from_bytes(raw[at:at + 4], "little")
        assert (word >> (16 * (j % 2) + 4 * (j // 2))) & 15 == codes[n, k]
        assert w.scales[t, k // group, r] == scales[n, k // group] and w.zeros[t, k // group, r] == zeros[n, k // group]
    want = (codes.float() - zeros.float().repeat_interleave(64, 1)[:, :K]) * scales.repeat_interleave(64, 1)[:, :K]
    assert torch.equal(ops.unpack_w4(w), want)


def test_pairs():
    from nkilab import ops

    a, b = (ops.quantize_w4(torch.randn(20, 128), 64) for _ in range(2))
    p = ops.pair_w4(a, b)
    assert p.paired and torch.equal(p.packed[0::2], a.packed) and torch.equal(p.scales[1::2], b.scales)
    for other in (ops.quantize_w4(torch.randn(20, 128), 32), ops.quantize_w4(torch.randn(21, 128), 64),
                  ops.quantize_w4(torch.randn(20, 128), 64, zeros=True),
                  ops.quantize_w4(torch.randn(20, 128), 64, scale_dtype=torch.float16)):
        with pytest.raises(ValueError):
            ops.pair_w4(a, other)
    with pytest.raises(ValueError):
        ops.pair_w4(p, p)
    with pytest.raises(ValueError):
        ops.unpack_w4(p)


def test_pack_refuses():
    from nkilab import ops

    c, s = torch.zeros(8, 256, dtype=torch.uint8), torch.ones(8, 2)
    for bad in (dict(codes=c.int()), dict(codes=c[0]), dict(codes=c[:0]), dict(scales=s[:, :1]), dict(group=100),
                dict(group=16), dict(group=64), dict(codes=c + 16), dict(zeros=torch.zeros(8, 2)),
                dict(zeros=torch.full((8, 2), 16, dtype=torch.uint8)), dict(zeros=torch.zeros(8, 1, dtype=torch.uint8))):
        kw = dict(codes=c, scales=s, group=128)
        kw.update(bad)
        with pytest.raises(ValueError):
            ops.pack_w4(**kw)
    with pytest.raises(TypeError):
        ops.pack_w4(c, s.double())
    with pytest.raises(ValueError):
        ops.quantize_w4(torch.randn(4, 64), 48)


def test_linear_refuses():
    from nkilab import ops

    w = ops.quantize_w4(torch.randn(20, 128), 64)
    a, c = torch.zeros(3, 128), torch.zeros(3, 20)
    for bad in (dict(a=a[:, :64]), dict(c=c[:2]), dict(c=torch.zeros(20, 3).t()), dict(residual=c[:2]),
                dict(residual=c.half()), dict(a=a[0])):
        kw = dict(a=a, w=w, c=c)
        kw.update(bad)
        with pytest.raises(ValueError):
            ops.linear_w4_into(**kw)
    with pytest.raises(TypeError):  # fp32 activations, 16-bit output
        ops.linear_w4_into(a, w, c.half())
    with pytest.raises(TypeError):  # fp16 scales, bf16 activations
        ops.linear_w4_into(a.bfloat16(), ops.quantize_w4(torch.randn(20, 128), 64, scale_dtype=torch.float16), c.bfloat16())
    with pytest.raises(ValueError, match="pair"):
        ops.linear_w4_into(a, ops.pair_w4(w, w), c)
    with pytest.raises(ValueError, match="pair"):
        ops.linear_w4_swiglu_into(a, w, c)
    with pytest.raises(ValueError, match="current device"):
        ops.linear_w4_into(a, w, c)


def test_abi_refusals():
    from nkilab import _lib

    def call(x=P, w=P, s=P, z=None, y=P, r=None, M=2, N=32, K=128, group=64, ldx=128, ldy=32, ldr=32, glu=0, dt=1, ds=1, do=1):
        return _lib.lib().nkl_gemm_w4(x, w, s, z, y, r, M, N, K, group, ldx, ldy, ldr, glu, dt, ds, do, None)

    for bad in (dict(M=-1), dict(N=-1), dict(K=-1), dict(K=0), dict(group=0), dict(group=48), dict(group=192), dict(ldx=127),
                dict(ldy=31), dict(r=P, ldr=31), dict(r=P, glu=1), dict(x=None), dict(w=None), dict(s=None), dict(y=None),
                dict(w=P + 8), dict(s=P + 8), dict(z=P + 4), dict(x=P + 1), dict(y=P + 1), dict(M=1 << 21, ldx=128),
                dict(M=1, ldx=-1)):
        assert call(**bad) == -1, bad
    for bad in (dict(dt=3), dict(ds=2), dict(do=2), dict(dt=0, ds=1, do=0), dict(dt=0, ds=0, do=1)):
        assert call(**bad) == -2, bad
    assert call(M=0, x=None, y=None) == 0 and call(N=0, ldy=0, y=None) == 0


def test_weight_refuses():
    """A W4Weight put together by hand (from a file, say) is checked as the kernels rely on it."""
    from nkilab import ops

    w = ops.quantize_w4(torch.randn(20, 200), 64, zeros=True)
    kw = dict(packed=w.packed, scales=w.scales, zeros=w.zeros, n=20, k=200, group=64)
    assert ops.W4Weight(**kw).n == 20
    for bad in (dict(packed=w.packed[:1]), dict(packed=w.packed.long()), dict(scales=w.scales[:, :2]), dict(zeros=w.zeros.int()),
                dict(zeros=w.zeros[:1]), dict(n=33), dict(k=300), dict(group=32), dict(group=96), dict(paired=True),
                dict(scales=w.scales.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            ops.W4Weight(**{**kw, **bad})
    with pytest.raises(TypeError):
        ops.W4Weight(**{**kw, "scales": w.scales.double()})


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_refuses_what_has_no_scale(zeros):
    """Infinities, NaN, and magnitudes whose scale leaves its type's range."""
    from nkilab import ops

    for x in (float("inf"), float("nan")):
        w = torch.ones(4, 128)
        w[2, 7] = x
        with pytest.raises(ValueError, match="finite"):
            ops.quantize_w4(w, zeros=zeros)
    big = torch.full((1, 128), 2e6)
    with pytest.raises(ValueError, match="finite"):
        ops.quantize_w4(big, zeros=zeros, scale_dtype=torch.float16)
    w = ops.quantize_w4(big, zeros=zeros, scale_dtype=torch.float32)
    assert (w.scales[0, 0, 0] - (2e6 / 15 if zeros else 2e6 / 7)).abs() <= 2e6 * 2.0 ** -23
