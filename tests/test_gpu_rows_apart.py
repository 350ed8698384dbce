"""Outputs in columns of the rows that inputs are columns of: they share no element, and are written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_rotation_between_columns():
    from nkilab import ops

    S, H, d = 33, 3, 64
    rows = torch.randn(S, 4 * H * d, generator=torch.Generator().manual_seed(0)).cuda()
    keep, r = rows.clone(), ops.Rotary(48, interleaved=True)
    part = lambda t, i: t[:, i * H * d:(i + 1) * H * d].view(S, H, d).transpose(0, 1)  # noqa: E731
    ops.rotary_into(part(rows, 2), part(rows, 1), r)
    assert torch.equal(part(rows, 1), ops.rotary(part(keep, 2), r))
    for i in (0, 2, 3):
        assert torch.equal(part(rows, i), part(keep, i))
    # heads in turn: x's and y's lie between each other
    x, y = (rows.view(S, 4 * H, d)[:, i::2].transpose(0, 1) for i in (0, 1))
    want = ops.rotary(x, r)
    ops.rotary_into(x, y, r)
    assert torch.equal(y, want)
    with pytest.raises(ValueError, match="share memory"):
        ops.rotary_into(part(rows, 1), rows[:, 2 * d:(2 + H) * d].view(S, H, d).transpose(0, 1), r)


def test_product_between_columns():
    from nkilab import ops

    g = torch.Generator().manual_seed(1)
    w = ops.quantize_w4(torch.randn(40, 128, generator=g).cuda(), 64)
    rows = torch.randn(70, 300, generator=g).cuda()
    keep = rows.clone()
    ops.linear_w4_into(rows[:, 100:228], w, rows[:, 50:90], residual=rows[:, 230:270])
    assert torch.equal(rows[:, 50:90], ops.linear_w4_into(keep[:, 100:228], w, torch.empty(70, 40, device="cuda"),
                                                          residual=keep[:, 230:270]))
    rows[:, 50:90] = keep[:, 50:90]
    assert torch.equal(rows, keep)
    for x, y, r in ((rows[:, :128], rows[:, 100:140], None), (rows[:, :128], rows[:, 128:168], rows[:, 129:169]),
                    (rows[:, :128], rows[1:, 100:140], None)):
        with pytest.raises(ValueError, match="share memory"):
            ops.linear_w4_into(x[:y.shape[0]], w, y, residual=r)


def test_append_with_q_between_columns():
    """q's columns rotated into others of the projection's rows, beside k's and v's."""
    from nkilab import ops

    B, H, Hkv, d = 5, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(B, (2 * H + 2 * Hkv) * d, generator=g).to(torch.bfloat16).cuda()
    part = lambda a, n: rows[:, a * d:(a + n) * d].view(B, n, d)  # noqa: E731
    q, k, v, out = part(0, H), part(H, Hkv), part(H + Hkv, Hkv), part(H + 2 * Hkv, H)
    kc, vc = (torch.zeros(B, Hkv, 16, d, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(B, Hkv, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1)
    lens = torch.full((B,), 7, dtype=torch.int32, device="cuda")
    r, keep = ops.Rotary(d), q.clone()
    ops.cache_append_into(k, v, kc, vc, table, lens, q=q, q_out=out, rotary=r, k_scale=ks, v_scale=vs)
    assert torch.equal(out, ops.rotary(keep.transpose(0, 1), r, positions=torch.full((B,), 6)).transpose(0, 1))
    assert torch.equal(q, keep)
    with pytest.raises(ValueError, match="share memory"):
        ops.cache_append_into(k, v, kc, vc, table, lens, q=q, q_out=part(H - 1, H), rotary=r, k_scale=ks, v_scale=vs)
