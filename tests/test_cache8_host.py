"""The 8-bit cache's reference against torch's type, and what its entry points refuse, with no GPU."""
import ctypes

import numpy as np
import pytest
import torch

import cache8_reference as R8
from test_paged_host import desc

P = 1 << 20


def test_reference_is_the_type():
    """Codes, their values and their rounding are torch.float8_e4m3fn's."""
    codes = torch.arange(256, dtype=torch.uint8)
    v = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(v, R8.NUM, equal_nan=True)
    x = torch.randn(20000, generator=torch.Generator().manual_seed(0)) * torch.logspace(-4, 2, 20000)
    x = torch.cat((x.clamp(-448, 448), torch.from_numpy(np.concatenate((R8.MID, -R8.MID))).float()))
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert R8.same(R8.encode(x.double().numpy()), want).all()
    assert [R8.scale_of(t) for t in (0.0, 448.0, 448.0001, 1e-30, 3e38)] == [17, 127, 128, 19, 246]


def d8(**kw):
    f = dict(dtype=3, k_row=64, d=64)
    f.update(kw)
    return desc(**f)


def scales(**kw):
    from nkilab import _lib

    f = dict(k=P, v=P, k_page=4, k_head=1, v_page=4, v_head=1)
    f.update(kw)
    return _lib.pack_scales(f["k"], f["v"], f["k_page"], f["k_head"], f["v_page"], f["v_head"])


def test_write_refuses():
    from nkilab import _lib, ops

    r = ops.Rotary(64)._packed

    def call(d=None, s=scales(), k=P, v=P, st=(256, 64, 256, 64), q=None, qo=None, H=0, sq=(0, 0, 0, 0), tree=None, words=0,
             rotary=None, dtype=1):
        return _lib.lib().nkl_cache_write(ctypes.byref(d or d8()), s, k, v, *st, q, qo, H, *sq, tree, words, rotary, dtype, None)

    for bad in (dict(s=None), dict(s=scales(k=0)), dict(s=scales(k_page=-1)), dict(k=None), dict(v=None),
                dict(st=(-256, 64, 256, 64)), dict(q=P, qo=P, H=4, sq=(256, 64, 256, 64)), dict(H=4, rotary=r),
                dict(q=P, rotary=r), dict(q=P, qo=P, H=4, sq=(256, 64, 512, 64), rotary=r), dict(tree=P),
                dict(rotary=ops.Rotary(128)._packed), dict(d=d8(d=56)), dict(d=d8(k_row=72)), dict(d=d8(k=P + 8)),
                dict(d=d8(table=None)), dict(d=d8(batch=-1)), dict(d=d8(lens=None))):
        assert call(**bad) == -1, bad
    assert call(dtype=3) == -2 and call(d=desc(dtype=2), dtype=1) == -2 and call(d=desc(dtype=7)) == -2
    assert call(d=d8(batch=0, rows=0, max_new=0)) == 0


def test_accept8_refuses():
    from nkilab import _lib

    def call(d=None, s=scales(), paths=P, row=4, cols=4, out=P + 4096, layers=2, st=(65536, 65536, 64, 64)):
        return _lib.lib().nkl_cache_accept8(ctypes.byref(d or d8()), s, paths, row, cols, out, layers, *st, None)

    for bad in (dict(s=None), dict(paths=None), dict(out=None), dict(cols=-1), dict(cols=1025), dict(layers=-1),
                dict(st=(65537, 65536, 64, 64)), dict(st=(65536, 65536, -1, 64)), dict(d=d8(d=24)), dict(d=d8(lens=None)),
                dict(d=d8(table=None)), dict(out=P)):
        assert call(**bad) == -1, bad
    assert call(d=desc()) == -2
    assert call(d=d8(batch=0, rows=0)) == 0


def test_attention8_refuses():
    from nkilab import _lib

    L = _lib.lib()

    def call(d=None, s=scales(), dtype=1, q=P, o=P, H=8, st=(512, 64, 512, 64), window=0, sinks=0, scale=0.125, ws=None, nb=0):
        return L.nkl_paged_attention8(ctypes.byref(d or d8()), s, dtype, q, o, H, *st, window, sinks, None, 0, scale, ws, nb, None)

    for bad in (dict(s=None), dict(s=scales(v=0)), dict(s=scales(v_head=-1)), dict(d=d8(d=72)), dict(d=d8(k_row=72)),
                dict(d=d8(d=144)), dict(st=(512, 64, 511, 64)), dict(H=6), dict(scale=0.0), dict(window=-1), dict(q=None)):
        assert call(**bad) == -1, bad
    assert call(dtype=3) == -2 and call(d=desc()) == -2
    assert L.nkl_paged_attention(ctypes.byref(d8()), P, P, 8, 512, 64, 512, 64, 0, 0, None, 0, 0.1, None, 0, None) == -2
    long = d8(table_cols=1000)
    n = L.nkl_paged_attention8_workspace_bytes(ctypes.byref(long), 8, 0, 0, 0, 1)
    assert n > 0 and call(d=long) == -4 and call(d=long, ws=P, nb=n - 1) == -4
    assert L.nkl_paged_attention8_workspace_bytes(ctypes.byref(desc(table_cols=1000)), 8, 0, 0, 0, 1) == 0


def test_operators_refuse():
    from nkilab import ops

    f8 = torch.zeros(4, 2, 16, 64, dtype=torch.float8_e4m3fn)
    sc = torch.zeros(4, 2, dtype=torch.uint8)
    bf = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    k, q = torch.zeros(2, 2, 64), torch.zeros(2, 4, 64)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    r = ops.Rotary(64)
    append = lambda kc=f8, **kw: ops.cache_append_into(k, k, kc, kc, table, lens, **kw)  # noqa: E731
    attend = lambda kc=f8, **kw: ops.paged_attention(q, kc, kc, table, lens, **kw)  # noqa: E731
    both = dict(k_scale=sc, v_scale=sc)
    for call in (append, attend, lambda kc=f8, **kw: ops.cache_copy_pages(kc, kc, [(0, 1)], **kw)):
        for bad in (dict(), dict(k_scale=sc), dict(v_scale=sc), dict(k_scale=sc.int(), v_scale=sc), dict(k_scale=sc[:3], v_scale=sc),
                    dict(k_scale=sc, v_scale=sc[None])):
            with pytest.raises(ValueError, match="scale"):
                call(**bad)
        with pytest.raises(ValueError, match="scales belong"):
            call(bf, **both)
        with pytest.raises(ValueError, match="current device"):
            call(**both)
    with pytest.raises(ValueError, match="either"):
        append(rope_base=100.0, rotary=r, **both)
    with pytest.raises(ValueError, match="go together"):
        append(q=q, q_out=q, **both)
    with pytest.raises(TypeError):
        append(bf)
    with pytest.raises(ValueError, match="scale"):
        ops.cache_accept(f8, f8, table, lens, table, n_nodes=1)


def test_cache_has_scales():
    from nkilab.cache import PagedCache

    c = PagedCache(5, 2, 64, layers=3, page_size=16, dtype=torch.float8_e4m3fn, device="cpu")
    assert c.k_scale.shape == c.v_scale.shape == (3, 5, 2) and c.k_scale.dtype is torch.uint8
    assert PagedCache(5, 2, 64, device="cpu").k_scale is None


def test_write_refuses_far_rows():
    """Row strides that the kernels' 32-bit row offsets cannot hold."""
    from nkilab import _lib, ops

    r = ops.Rotary(64)._packed
    for st, sq in (((1 << 31, 64, 256, 64), (256, 64, 256, 64)), ((256, 64, 1 << 31, 64), (256, 64, 256, 64)),
                   ((256, 64, 256, 64), (1 << 31, 64, 256, 64)), ((256, 64, 256, 64), (256, 64, 1 << 31, 64))):
        assert _lib.lib().nkl_cache_write(ctypes.byref(d8()), scales(), P, P, *st, P, P, 4, *sq, None, 0, r, 1, None) == -1


def test_writes_refuse_shared_scales():
    """Exponents that pages, heads, layers, or K and V share; rows of q_out in one place."""
    from nkilab import _lib, ops

    L = _lib.lib()
    r = ops.Rotary(64)._packed
    apart = dict(v=P + 4096)

    def write(s, so=(256, 64)):
        return L.nkl_cache_write(ctypes.byref(d8()), s, P, P, 256, 64, 256, 64, P, P + 64, 4, 256, 64, *so, None, 0, r, 1, None)

    for bad in (dict(v=P), dict(k_page=0), dict(v_page=0), dict(k_head=0), dict(v_head=0)):
        s = scales(**{**apart, **bad})
        assert write(s) == -1 and b"share scales" in L.nkl_last_error_string(), bad
        assert L.nkl_cache_accept8(ctypes.byref(d8()), s, P, 4, 4, P + 256, 2, 16, 16, 16, 16, None) == -1, bad
        assert b"share scales" in L.nkl_last_error_string()
    for so in ((0, 64), (256, 0)):
        assert write(scales(**apart), so) == -1 and b"share memory" in L.nkl_last_error_string()
    for layers in ((0, 16), (16, 0)):
        assert L.nkl_cache_accept8(ctypes.byref(d8()), scales(**apart), P, 4, 4, P + 256, 2, 16, 16, *layers, None) == -1
        assert b"layers share" in L.nkl_last_error_string()
