"""What the paged cache's entry points refuse, checked with no GPU, and what
their plans say of sizes."""
import ctypes

import numpy as np
import pytest
import torch

P = 1 << 20  # (an aligned address, refused before it is used)


def desc(**kw):
    from nkilab import _lib

    f = dict(k=P, v=P, k_page=4096, k_head=1024, k_row=64, v_page=4096, v_head=1024, v_row=64, table=P, table_row=8, lens=P,
             q_start=None, pages=10, kv_heads=4, page_size=16, d=64, table_cols=8, batch=2, rows=2, max_new=1, dtype=1)
    f.update(kw)
    return _lib.PagedCacheDesc(*(f[n] for n, _ in _lib.PagedCacheDesc._fields_))


def test_packed_description():
    """The bytes that the operators pass are the structure, field for field."""
    from nkilab import _lib

    values = list(range(1, len(_lib.PagedCacheDesc._fields_) + 1))
    packed, d = _lib.pack_cache(*values), _lib.PagedCacheDesc(*values)
    assert packed == bytes(d)[:len(packed)] and 0 <= ctypes.sizeof(d) - len(packed) < 8
    # (the library reads the whole structure; what may be missing at its end is padding)
    assert _lib.PagedCacheDesc.dtype.offset + 4 == len(packed)


def attn(d, q=P, o=P, H=8, st=(512, 64, 512, 64), window=0, sinks=0, tree=None, words=0, scale=0.125, ws=None, nb=0):
    from nkilab import _lib

    return _lib.lib().nkl_paged_attention(ctypes.byref(d), q, o, H, *st, window, sinks, tree, words, scale, ws, nb, None)


def test_paged_attention_abi_refusals():
    from nkilab import _lib

    assert attn(desc(dtype=7)) == -2
    for bad in (dict(batch=-1), dict(pages=-1), dict(page_size=0), dict(d=136), dict(d=60), dict(kv_heads=3),
                dict(rows=3), dict(lens=None), dict(k_row=-64), dict(k_row=66), dict(v=P + 8), dict(table_cols=1 << 27),
                dict(table=None), dict(batch=70000, rows=70000)):
        assert attn(desc(**bad)) == -1, bad
    for bad in (dict(H=0), dict(H=6), dict(window=-1), dict(sinks=-2), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(tree=P, words=0), dict(q=None), dict(o=P + 2), dict(st=(512, 64, 511, 64))):
        assert attn(desc(), **bad) == -1, bad
    assert b"" != _lib.lib().nkl_last_error_string()
    assert _lib.lib().nkl_paged_attention(None, P, P, 8, 0, 0, 0, 0, 0, 0, None, 0, 1.0, None, 0, None) == -1
    # nothing to do
    assert attn(desc(batch=0, rows=0, max_new=0), q=None, o=None) == 0
    # a long table needs a workspace, and one that is too small is refused before a launch
    d = desc(table_cols=1000)
    n = _lib.lib().nkl_paged_attention_workspace_bytes(ctypes.byref(d), 8, 0, 0, 0)
    assert n > 0 and attn(d) == -4 and attn(d, ws=P, nb=n - 1) == -4 and attn(d, ws=P + 4, nb=n) == -1
    # a short window needs none, nor does a batch that fills the card
    assert _lib.lib().nkl_paged_attention_workspace_bytes(ctypes.byref(d), 8, 64, 0, 0) == 0
    big = desc(table_cols=1000, batch=4096, rows=4096)
    assert _lib.lib().nkl_paged_attention_workspace_bytes(ctypes.byref(big), 8, 0, 0, 0) == 0


def test_mover_abi_refusals():
    from nkilab import _lib

    L = _lib.lib()

    def append(d, k=P, v=P, q=None, qo=None, H=0, tree=None, words=0, base=0.0):
        return L.nkl_cache_append(ctypes.byref(d), k, v, 256, 64, 256, 64, q, qo, H, 512, 64, 512, 64, tree, words, base, None)

    assert append(desc(batch=0, rows=0, max_new=0)) == 0
    for d, kw in ((desc(rows=3), {}), (desc(), dict(k=None)), (desc(), dict(base=1.0)), (desc(), dict(base=-3.0)),
                  (desc(), dict(base=float("inf"))), (desc(d=63), dict(base=100.0)), (desc(), dict(q=P, qo=P, H=8)),
                  (desc(), dict(q=P, qo=None, H=8, base=100.0)), (desc(), dict(H=8, base=100.0)),
                  (desc(max_new=65, rows=130), dict(tree=P, words=1)), (desc(table=None), {})):
        assert append(d, **kw) == -1, kw

    def copy(pairs, d=None, layers=1, n=None):
        a = np.array(pairs, np.int32).reshape(-1, 2)
        return L.nkl_cache_copy_pages(ctypes.byref(d or desc()), a.ctypes.data, len(a) if n is None else n, layers, 0, 0, None)

    assert copy([]) == 0 and copy([(0, 1)], layers=0) == 0
    for pairs in ([(0, 10)], [(-1, 2)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)], [(1, 2), (0, 1)]):
        assert copy(pairs) == -1, pairs
    assert copy([(0, 1)], n=-1) == -1 and copy([(0, 1)], layers=40000) == -1 and copy([(0, 1)], d=desc(k=None)) == -1

    def accept(d, paths=P, row=4, cols=4, new=P, layers=1):
        return L.nkl_cache_accept(ctypes.byref(d), paths, row, cols, new, layers, 0, 0, None)

    assert accept(desc(batch=0, rows=0)) == 0
    for d, kw in ((desc(), dict(cols=-1)), (desc(), dict(paths=None)), (desc(), dict(new=None)), (desc(), dict(layers=-1)),
                  (desc(table=None, batch=1, rows=1), {}), (desc(lens=None), {}), (desc(batch=70000, rows=70000), {})):
        assert accept(d, **kw) == -1, kw
    assert L.nkl_tree_mask(P, None, 2, 5, 2, P, 1, None) == -1 and L.nkl_tree_mask(None, None, 1, 5, 5, P, 1, None) == -1
    assert L.nkl_tree_mask(P, None, 1, 5, 5, P, 0, None) == -1 and L.nkl_tree_mask(None, None, 0, 0, 0, None, 1, None) == 0


def tensors(**kw):
    t = dict(q=torch.zeros(2, 8, 64), k_cache=torch.zeros(10, 4, 16, 64), v_cache=torch.zeros(10, 4, 16, 64),
             page_table=torch.zeros(2, 5, dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32))
    t.update(kw)
    return t


def test_paged_attention_refusals():
    from nkilab import ops

    call = lambda **kw: ops.paged_attention(**tensors(**kw))  # noqa: E731
    for kw in (dict(q=torch.zeros(2, 8, 32)), dict(q=torch.zeros(2, 6, 64)), dict(q=torch.zeros(3, 8, 64)),
               dict(k_cache=torch.zeros(9, 4, 16, 64)), dict(page_table=torch.zeros(2, 5, dtype=torch.int64)),
               dict(page_table=torch.zeros(10, dtype=torch.int32)), dict(lens=torch.zeros(3, dtype=torch.int32)),
               dict(lens=torch.zeros(2)), dict(q_start=torch.zeros(3, dtype=torch.int32)),
               dict(q_start=torch.zeros(2, dtype=torch.int32), max_q=1), dict(max_q=2), dict(window=0), dict(sinks=3),
               dict(window=4, sinks=-1), dict(tree=torch.zeros(2, 1, dtype=torch.int32)),
               dict(tree=torch.zeros(3, 1, dtype=torch.int64)), dict(tree=torch.zeros(2, 0, dtype=torch.int64)),
               dict(k_cache=torch.zeros(10, 4, 64, 16).transpose(2, 3))):
        with pytest.raises(ValueError) as e:
            call(**kw)
        assert "current device" not in str(e.value), (kw, e.value)  # (refused for what it is)
    with pytest.raises(TypeError):
        call(q=torch.zeros(2, 8, 64).bfloat16())
    with pytest.raises(ValueError, match="current device"):  # CPU tensors
        call()


def test_mover_refusals():
    from nkilab import ops

    t = tensors()
    kc, vc, table, lens = t["k_cache"], t["v_cache"], t["page_table"], t["lens"]
    k = torch.zeros(2, 4, 64)
    q = torch.zeros(2, 8, 64)
    for args, kw in (((k[:, :3], k[:, :3]), {}), ((k, k[:1]), {}), ((k, k), dict(q=q)), ((k, k), dict(q=q, q_out=q)),
                     ((k, k), dict(q=q[:1], q_out=q[:1], rope_base=1e4)), ((k, k), dict(rope_base=0.5)),
                     ((k, k), dict(q=q, q_out=q[:, :4], rope_base=1e4))):
        with pytest.raises(ValueError) as e:
            ops.cache_append_into(*args, kc, vc, table, lens, **kw)
        assert "current device" not in str(e.value), kw
    with pytest.raises(TypeError):
        ops.cache_append_into(k.half(), k.half(), kc, vc, table, lens)
    for pairs in ([(0, 10)], [(-1, 0)], [1, 2], [(0.5, 1.0)]):
        with pytest.raises(ValueError) as e:
            ops.cache_copy_pages(kc, vc, pairs)
        assert "current device" not in str(e.value), pairs
    ops.cache_copy_pages(kc, vc, [])
    paths = torch.zeros(2, 3, dtype=torch.int32)
    for args, kw in (((paths,), {}), ((paths[:1],), dict(n_nodes=3)), ((paths.long(),), dict(n_nodes=3)),
                     ((paths,), dict(n_nodes=-1)), ((paths,), dict(n_nodes=3, q_start=lens))):
        with pytest.raises(ValueError) as e:
            ops.cache_accept(kc, vc, table, lens, *args, **kw)
        assert "current device" not in str(e.value), kw
    for kw in (dict(batch=2), dict(q_start=lens), dict(max_q=4)):
        with pytest.raises(ValueError) as e:
            ops.tree_mask(torch.zeros(5, dtype=torch.int32), **kw)
        assert "current device" not in str(e.value), kw
