"""Steps of no rows, and other smallest calls of the decoder over a cache, on the GPU."""
import pytest
import torch

from test_paged_cache import D, KV, HEADS, block_close, make_block, make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [None, 5])
def test_steps_of_no_rows(dtype, window):
    """A step in which no sequence brings a row leaves the cache as it is; one
    in which some bring none gives the others theirs."""
    from nkilab.model import nki_decode

    block, cache = make_block(window), make_cache(dtype)
    a, b = cache.add(), cache.add()
    run = lambda x, step: nki_decode(block, x.cuda(), cache, step, compute_dtype=dtype).cpu()  # noqa: E731
    for seqs, counts, tree in (([], [], None), ([a, b], [0, 0], None), ([a, b], [0, 0], [[], []])):
        assert run(torch.zeros(0, D), cache.step(seqs, counts, tree)).shape == (0, D)
    x = torch.randn(9, D)
    out = [run(x[:1], cache.step([a, b], [0, 1]))]
    bits = lambda: [t.view(torch.uint8).clone() for t in (cache.k, cache.v)]  # noqa: E731  (rows never written may be NaN)
    held = bits()
    step = cache.step([a, b], [0, 0])
    run(torch.zeros(0, D), step)
    cache.accept(step, [[], []])
    assert all(map(torch.equal, held, bits())) and cache.length(b) == 1
    out += [run(x[1:8], cache.step([b, a], [7, 0])), run(x[8:], cache.step([a, b], [0, 1], [[], [-1]]))]
    block_close(torch.cat(out), block(x).detach(), dtype)


def test_operators_on_no_rows():
    from nkilab import ops

    hd = D // HEADS
    kc = torch.randn(4, KV, 16, hd, device="cuda")
    vc = kc.clone()
    i32 = dict(dtype=torch.int32, device="cuda")
    none = torch.empty(0, KV, hd, device="cuda")
    q = torch.empty(0, HEADS, hd, device="cuda")
    for B in (0, 2):
        table, lens, starts = torch.zeros(B, 1, **i32), torch.full((B,), 3, **i32), torch.zeros(B + 1, **i32)
        ops.cache_append_into(none, none, kc, vc, table, lens, q_start=starts, max_q=0, q=q, q_out=q, rope_base=1e4)
        assert ops.paged_attention(q, kc, vc, table, lens, q_start=starts, max_q=0).shape == q.shape
        got = ops.cache_accept(kc, vc, table, lens, torch.zeros(B, 0, **i32), q_start=starts)
        assert torch.equal(got, lens)
        words = ops.tree_mask(torch.empty(0, **i32), q_start=starts, max_q=0, window=3, sinks=1, lens=lens)
        assert words.shape == (0, 1)
    assert torch.equal(kc, vc)
