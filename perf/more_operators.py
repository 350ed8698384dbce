"""Operators of decoding in few bits, as cases that can be timed and checked.

Rotary positions in both layouts, over part of a head, with frequencies scaled
for long contexts; products with 4-bit weights and group scales; and a paged
cache of 8-bit K and V rows with a power-of-two scale for each page and head:
new rows written to it (rotated on the way), and attention over it.

``own`` selects what ``run`` calls: the operators' plain form in torch, or the
framework's entry points.  ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
SCALE_BIAS = 127            # a scale byte s stands for 2^(s - 127)
SCALE_LO, SCALE_HI = 17, 246  # the scale bytes that appended rows get
BASE = 10000.0


def _ops():
    pkg = os.path.abspath("nki-kernel-lab_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from nkilab import ops

    return ops


# ---------------------------------------------------------------- cases --

def _rotary(name, H, S, d, rot, interleaved, scaling, factor, original, far, grad, dtype):
    return {"name": name, "op": "rotary", "H": H, "S": S, "d": d, "rot": rot, "interleaved": interleaved, "scaling": scaling,
            "factor": factor, "original": original, "far": far, "grad": grad, "dtype": dtype}


def _linear(name, M, N, K, group, zeros, glu, residual, dtype):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "group": group, "zeros": zeros, "glu": glu,
            "residual": residual, "dtype": dtype}


def _append(name, B, n_lo, n_hi, len_lo, len_hi, H, Hkv, d, page, rot, interleaved, dtype):
    return {"name": name, "op": "append", "B": B, "n_lo": n_lo, "n_hi": n_hi, "len_lo": len_lo, "len_hi": len_hi, "H": H,
            "Hkv": Hkv, "d": d, "page": page, "rot": rot, "interleaved": interleaved, "dtype": dtype}


def _attend(name, B, n_lo, n_hi, len_lo, len_hi, H, Hkv, d, page, window, sinks, tree, dtype):
    return {"name": name, "op": "attend", "B": B, "n_lo": n_lo, "n_hi": n_hi, "len_lo": len_lo, "len_hi": len_hi, "H": H,
            "Hkv": Hkv, "d": d, "page": page, "window": window, "sinks": sinks, "tree": tree, "dtype": dtype}


def listed():
    return [
        # One new token for each of 64 running sequences, Q and K heads together: a decode step's, where latency counts.
        _rotary("rotary_step", 40, 64, 128, 128, False, "none", 1.0, 0, 10000, False, "bf16"),
        # A long prompt's Q and K, half of each head rotated in the interleaved layout, for a context stretched eightfold.
        _rotary("rotary_prompt", 40, 8192, 128, 64, True, "bands", 8.0, 8192, 131072, False, "fp16"),
        # The gradient of the decoder block's q in fp32, stretched frequencies with their magnitude.
        _rotary("rotary_grad", 16, 2048, 128, 128, False, "parts", 16.0, 4096, 65536, True, "fp32"),
        # One token through the decoder block's output projection: the smallest product.
        _linear("linear_token", 1, 2048, 2048, 128, False, False, True, "bf16"),
        # Sixteen sequences' tokens through the gate and up projections.
        _linear("linear_batch", 16, 5632, 2048, 128, True, True, False, "fp16"),
        # Drafted tokens through sizes off every tile, fp32 activations, small groups.
        _linear("linear_odd", 77, 1001, 1990, 32, True, False, False, "fp32"),
        # The decoder block's prompt through the gate and up projections: bound by the matrix cores.
        _linear("linear_prompt", 2048, 5632, 2048, 64, False, True, False, "bf16"),
        # One new token for each of 64 running sequences into the cache.
        _append("append8_step", 64, 1, 1, 100, 1000, 32, 8, 128, 64, 128, False, "bf16"),
        # Ragged prompts and chunks of prompts enter the cache.
        _append("append8_prompts", 6, 700, 2048, 700, 3500, 16, 16, 128, 64, 64, True, "fp16"),
        # One token each for a ragged batch over long caches: a decode step's attention, the largest cache.
        _attend("attend8_decode", 64, 1, 1, 200, 16384, 32, 8, 128, 64, 0, 0, False, "bf16"),
        # Trees of drafted tokens for a few sequences with small pages.
        _attend("attend8_tree", 8, 24, 24, 500, 4000, 16, 4, 128, 16, 0, 0, True, "fp16"),
        # Chunks of prompts over what is cached of them, under a window with the first tokens kept.
        _attend("attend8_chunks", 4, 500, 2000, 2000, 8000, 32, 8, 128, 128, 4096, 4, False, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _strip(c):
    del c["name"]
    return c


def draw(rng):
    op = rng.choice(("rotary", "linear", "linear", "append", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "linear":
        M = rng.choice((1, _log(rng, 2, 64), _log(rng, 2, 64), _log(rng, 65, 2048)))
        N, K = _log(rng, 64, 12000), _log(rng, 64, 12000)
        while N * K > 2 ** 25 or M * N * K > 2 ** 34:
            N, K = N * 4 // 5, K * 4 // 5
        if rng.random() < 0.6:
            N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
        glu = rng.random() < 0.3
        return _strip(_linear("", M, N, K, rng.choice((32, 64, 128, 128, 256)), rng.random() < 0.5, glu,
                              not glu and rng.random() < 0.5, dtype))
    Hkv, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 4, 7, 8))
    if Hkv * group > 40:
        group = 40 // Hkv
    H = Hkv * group
    if op == "rotary":
        d = rng.choice((64, 80, 96, 128, 128, 256))
        S = _log(rng, 1, 16384)
        while (H + Hkv) * S * d * BYTES[dtype] > 2 ** 27:
            S = S // 2
        scaling = rng.choice(("none", "linear", "base", "parts", "bands"))
        return _strip(_rotary("", H + Hkv, S, d, rng.choice((d, d, d // 2, d // 4 * 2)), rng.random() < 0.5, scaling,
                              1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0, 32.0)),
                              rng.choice((2048, 4096, 8192)), _log(rng, 20000, 1000000), rng.random() < 0.3, dtype))
    d = rng.choice((32, 64, 64, 80, 96, 128, 128, 128))
    page = rng.choice((8, 16, 16, 24, 32, 64, 64, 100, 128, 256))
    if op == "append":
        n = rng.choice((1, 1, _log(rng, 2, 2000)))
        B = _log(rng, 1, 64 if n == 1 else 8)
        hi = n + _log(rng, 1, 2000)
        while B * hi * Hkv * d > 2 ** 26:
            B, hi = (B + 1) // 2, n + (hi - n) // 2
            if B == 1 and hi == n:
                break
        return _strip(_append("", B, max(1, n // 3), n, max(1, n // 2) + (hi - n) // 4, hi, H, Hkv, d, page,
                              rng.choice((0, d, d, d // 4 * 2)), rng.random() < 0.5, dtype))
    window = rng.choice((0, 0, _log(rng, 1, 8192), _log(rng, 64, 4096)))
    sinks = rng.choice((0, 1, 4, 16, 100)) if window else 0
    tree = rng.random() < 0.2
    n = _log(rng, 2, 128) if tree else rng.choice((1, 1, 1, _log(rng, 2, 500)))
    B = _log(rng, 1, 128 if n == 1 else 8)
    hi = n + _log(rng, 1, 30000 if n == 1 else 4000)
    while B * hi * Hkv * d > 2 ** 28 or B * n * hi * H > 2 ** 28:
        B, hi = (B + 1) // 2, n + (hi - n) * 3 // 4
    return _strip(_attend("", B, n if tree else max(1, n // 3), n, n + (hi - n) // 4, hi, H, Hkv, d, page, window, sinks,
                          tree, dtype))


def _spread(lo, hi, B):
    """B whole numbers from lo to hi, evenly spread."""
    return [hi] if B == 1 else [lo + (hi - lo) * b // (B - 1) for b in range(B)]


def _counts(case):
    """Rows of each sequence, new ones included, and its new rows; in the order of length."""
    lens = _spread(case["len_lo"], case["len_hi"], case["B"])
    return lens, [min(n, length) for n, length in zip(_spread(case["n_lo"], case["n_hi"], case["B"]), lens)]


# --------------------------------------------------------------- inputs --

def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(DTYPES[dtype])


def _parents(rng, n):
    """A drafted tree in the order it is drafted: each node hangs off an earlier one, the first off the context."""
    return [-1] + [rng.randrange(max(0, i - 12), i) for i in range(1, n)]


def _mask_words(parents, width):
    """Node i's ancestors and itself, as bits of ``width`` 64-bit words (held as int64)."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << i))
    signed = lambda w: w - (1 << 64) if w >> 63 else w  # noqa: E731
    return [[signed((r >> (64 * w)) & (2 ** 64 - 1)) for w in range(width)] for r in rows]


def _tables(rng, lens, page, spare):
    """A page table over randomly placed pages, -1 behind each sequence's last, and the pool's page count."""
    need = [-(-length // page) for length in lens]
    pool = list(range(sum(need) + spare))
    rng.shuffle(pool)
    width = max(need)
    rows, at = [], 0
    for c in need:
        rows.append(pool[at:at + c] + [-1] * (width - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), sum(need) + spare


def _cache(gen, pages, Hkv, page, d):
    """A cache of e4m3 codes, and its scale bytes: rows of a normal distribution, each page and head with a magnitude."""
    codes = torch.empty((pages, Hkv, page, d), dtype=E4M3, device="cuda")
    scales = torch.empty((pages, Hkv), dtype=torch.uint8, device="cuda")
    step = max(1, 2 ** 28 // (Hkv * page * d))
    for p in range(0, pages, step):
        x = torch.randn((min(step, pages - p), Hkv, page, d), generator=gen, device="cuda")
        x *= 0.5 + torch.rand((x.shape[0], Hkv, 1, 1), generator=gen, device="cuda")
        e = torch.ceil(torch.log2(x.abs().amax(dim=(2, 3)) / E4M3_MAX * 1.0001))
        codes[p:p + step] = (x * torch.exp2(-e)[:, :, None, None]).to(E4M3)
        scales[p:p + step] = (e + SCALE_BIAS).to(torch.uint8)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    st = {"case": case}
    dt = case["dtype"]
    if case["op"] == "rotary":
        H, S, d = case["H"], case["S"], case["d"]
        # (rows of a token together, as a projection writes them)
        st["x"] = _randn(gen, (S, H, d), dt).transpose(0, 1)
        st["y"] = torch.empty_like(st["x"])
        # A stretch of positions from somewhere below `far`, or one of its own for each row.
        if S > 200:
            first = rng.randrange(max(1, case["far"] - S))
            st["positions"] = torch.arange(first, first + S, dtype=torch.int32, device="cuda")
        else:
            st["positions"] = torch.tensor([rng.randrange(case["far"]) for _ in range(S)], dtype=torch.int32, device="cuda")
        if own:
            st["rotary"] = _ops().Rotary(case["rot"], BASE, interleaved=case["interleaved"],
                                         scaling=None if case["scaling"] == "none" else case["scaling"],
                                         factor=case["factor"], original=case["original"])
        return st
    if case["op"] == "linear":
        M, N, K, group = case["M"], case["N"], case["K"], case["group"]
        G = -(-K // group)
        st["x"] = _randn(gen, (M, K), dt)
        sides = 2 if case["glu"] else 1  # gate and up, or one weight
        st["codes"] = [torch.randint(0, 16, (N, K), generator=gen, device="cuda", dtype=torch.uint8) for _ in range(sides)]
        # Scales such that outputs are of the order of one.
        st["scales"] = [((0.5 + torch.rand((N, G), generator=gen, device="cuda")) / (4.6 * math.sqrt(K)))
                        .to(torch.float32 if dt == "fp32" else DTYPES[dt]) for _ in range(sides)]
        st["zeros"] = [torch.randint(5, 11, (N, G), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
                       for _ in range(sides)]
        st["residual"] = _randn(gen, (M, N), dt) if case["residual"] else None
        st["y"] = torch.empty((M, N), dtype=DTYPES[dt], device="cuda")
        if own:
            ops = _ops()
            parts = [ops.pack_w4(c, s, z, group) for c, s, z in zip(st["codes"], st["scales"], st["zeros"])]
            st["w"] = ops.pair_w4(*parts) if case["glu"] else parts[0]
        return st
    d, Hkv = case["d"], case["Hkv"]
    lens, news = _counts(case)
    order = list(range(case["B"]))
    rng.shuffle(order)
    lens, news = [lens[i] for i in order], [news[i] for i in order]
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    table, pages = _tables(rng, lens, case["page"], 3)
    kc, ks = _cache(gen, pages, Hkv, case["page"], d)
    vc, vs = _cache(gen, pages, Hkv, case["page"], d)
    st.update(kc=kc, vc=vc, ks=ks, vs=vs, table=table, lens_host=lens, news_host=news, starts_host=starts,
              lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
              q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_q=max(news), tree=None)
    T = starts[-1]
    st["q"] = _randn(gen, (T, case["H"], d), dt)
    if case["op"] == "append":
        st.update(k=_randn(gen, (T, Hkv, d), dt), v=_randn(gen, (T, Hkv, d), dt), q_out=torch.empty_like(st["q"]))
        # A few channels of keys are far larger than the others.
        st["k"][:, :, 1::29] *= 8
        st["rotary"] = None
        if own and case["rot"]:
            st["rotary"] = _ops().Rotary(case["rot"], BASE, interleaved=case["interleaved"])
    elif case["tree"]:
        width = -(-max(news) // 64)
        words = [w for n in news for w in _mask_words(_parents(rng, n), width)]
        st["tree"] = torch.tensor(words, dtype=torch.int64, device="cuda")
    return st


# ------------------------------------------------------------------ run --

def run(state):
    return _own(state) if own else _plain(state)


def _own(st):
    ops, case = _ops(), st["case"]
    if case["op"] == "rotary":
        return ops.rotary_into(st["x"], st["y"], st["rotary"], positions=st["positions"], grad=case["grad"])
    if case["op"] == "linear":
        if case["glu"]:
            return ops.linear_w4_swiglu_into(st["x"], st["w"], st["y"])
        return ops.linear_w4_into(st["x"], st["w"], st["y"], residual=st["residual"])
    if case["op"] == "append":
        q = st["q"] if case["rot"] else None
        ops.cache_append_into(st["k"], st["v"], st["kc"], st["vc"], st["table"], st["lens"], q_start=st["q_start"],
                              max_q=st["max_q"], q=q, q_out=st["q_out"] if case["rot"] else None, rotary=st["rotary"],
                              k_scale=st["ks"], v_scale=st["vs"])
        return (st["kc"], st["vc"], st["ks"], st["vs"]) + ((st["q_out"],) if case["rot"] else ())
    return ops.paged_attention(st["q"], st["kc"], st["vc"], st["table"], st["lens"], q_start=st["q_start"],
                               max_q=st["max_q"], window=case["window"] or None, sinks=case["sinks"], tree=st["tree"],
                               k_scale=st["ks"], v_scale=st["vs"])


def _frequencies(case, device):
    """Angles per position of the rotated pairs (64 bits), and the factor of the rotated elements."""
    rot, scaling, s = case["rot"], case.get("scaling", "none"), case.get("factor", 1.0)
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    if scaling == "base" and rot > 2:
        return (BASE * s ** (rot / (rot - 2))) ** (-2 * i / rot), 1.0
    f = BASE ** (-2 * i / rot)
    if scaling == "linear":
        return f / s, 1.0
    if scaling == "parts":
        index = lambda turns: rot * math.log(case["original"] / (2 * math.pi * turns)) / (2 * math.log(BASE))  # noqa: E731
        lo, hi = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / s * ramp, 0.1 * math.log(s) + 1
    if scaling == "bands":
        turns = case["original"] * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / s * (1 - keep), 1.0
    return f, 1.0


def _rotate(x, pos, case, sign=1.0, wide=torch.float32):
    """The first elements of rows x [T, heads, d] rotated by their positions [T]; `wide` bits."""
    rot = case["rot"]
    f, m = _frequencies(case, x.device)
    a = pos.double()[:, None, None] * f
    cos, sin = (m * torch.cos(a)).to(wide), (sign * m * torch.sin(a)).to(wide)
    y = x.to(wide).clone()
    if case["interleaved"]:
        x1, x2 = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2], y[..., 1:rot:2] = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    else:
        x1, x2 = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
        y[..., :rot // 2], y[..., rot // 2:rot] = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    return y


def _raw(codes):
    return codes.view(torch.uint8)


def _pick(codes, pages):
    return _raw(codes)[pages].view(E4M3)


def _power(e):
    """2^e, exactly (64 bits), for whole e."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _nearest_e4m3(x):
    """x (64 bits, within the type's range) rounded to e4m3, ties to even."""
    _, e = torch.frexp(x)
    step = _power(torch.clamp(e - 1, min=-6) - 3)
    return (torch.round(x / step) * step).to(E4M3)


def _scale_bytes(top):
    """The smallest scale whose range holds `top` (64 bits)."""
    m, e = torch.frexp(top / E4M3_MAX)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(top > 0, (e + SCALE_BIAS).clamp(SCALE_LO, SCALE_HI), torch.full_like(e, SCALE_LO))


def _write_rows(case, codes, scales, rows, page, within, first_page, first_row):
    """Rows (64 bits, [T, Hkv, d]) to places (page, within); sequences' first new rows at (first_page, first_row)."""
    size = case["page"]
    new = torch.zeros(scales.shape, dtype=torch.float64, device=rows.device)
    new.scatter_reduce_(0, page[:, None].expand(-1, case["Hkv"]), rows.abs().amax(dim=2), "amax")
    touched = torch.zeros(scales.shape[0], dtype=torch.bool, device=rows.device)
    touched[page] = True
    want = _scale_bytes(new)
    # Rows before the new ones keep their page's scale, and are brought to the new one where it is larger.
    kept = first_page[first_row > 0]
    old = scales[kept].to(want.dtype)
    want[kept] = torch.maximum(want[kept], old)
    shrink = _power(old - want[kept])[:, :, None, None]
    before = torch.arange(size, device=rows.device)[None, None, :, None] < first_row[first_row > 0][:, None, None, None]
    there = _pick(codes, kept).double()
    _raw(codes)[kept] = _raw(torch.where(before, _nearest_e4m3(there * shrink).double(), there).to(E4M3))
    scales[touched] = want[touched].to(torch.uint8)
    scale = _power(want[page] - SCALE_BIAS)
    _raw(codes)[page, :, within] = _raw(_nearest_e4m3((rows / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)))


def _values(codes, scales):
    """Rows [pages, Hkv, page, d] of codes by their scale bytes [pages, Hkv]; 32 bits."""
    return codes.float() * _power(scales.to(torch.int64) - SCALE_BIAS).float()[:, :, None, None]


def _row_slots(st, b, j):
    """Pages and offsets within them of rows j of sequence b."""
    page = st["case"]["page"]
    return st["table"][b].long()[j // page], j % page


def _softmax_rows(s, visible):
    s = s.masked_fill(~visible, float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _window(j, pos, window, sinks):
    """Keys j [L] that a query at pos [n] sees of those before it: [n, L]."""
    seen = j[None] <= pos[:, None]
    if window:
        seen &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
    return seen


def _tree_bits(words, n):
    """Mask words [n, W] as truth values [n, n]."""
    i = torch.arange(n, device=words.device)
    return ((words[:, i // 64] >> (i % 64)) & 1).bool()


def _attention(q, k, v, visible):
    """q [n, H, d], k, v [Hkv, L, d], visible [n, L]; 32 bits."""
    n, H, d = q.shape
    Hkv, L, _ = k.shape
    g = H // Hkv
    qf = q.float().view(n, Hkv, g, d).permute(1, 2, 0, 3).reshape(Hkv, g * n, d) / math.sqrt(d)
    s = torch.matmul(qf, k.transpose(1, 2).contiguous()).view(Hkv, g, n, L)
    p = _softmax_rows(s, visible).view(Hkv, g * n, L)
    return torch.matmul(p, v).view(Hkv, g, n, d).permute(2, 0, 1, 3).reshape(n, H, d)


def _dense(st, side):
    """One side's weight [N, K] in 32 bits."""
    group, K = st["case"]["group"], st["case"]["K"]
    spread = lambda t: t.float().repeat_interleave(group, dim=1)[:, :K]  # noqa: E731
    zeros = st["zeros"][side]
    return (st["codes"][side].float() - (8.0 if zeros is None else spread(zeros))) * spread(st["scales"][side])


def _plain(st):
    case = st["case"]
    if case["op"] == "rotary":
        y = _rotate(st["x"].transpose(0, 1), st["positions"], case, -1.0 if case["grad"] else 1.0)
        st["y"].copy_(y.transpose(0, 1))
        return st["y"]
    if case["op"] == "linear":
        x = st["x"].float()
        y = torch.matmul(x, _dense(st, 0).t())
        if case["glu"]:
            y = y / (1 + torch.exp(-y)) * torch.matmul(x, _dense(st, 1).t())
        if st["residual"] is not None:
            y = y + st["residual"].float()
        st["y"].copy_(y)
        return st["y"]
    if case["op"] == "append":
        pos = torch.cat([torch.arange(length - n, length, device="cuda")
                         for length, n in zip(st["lens_host"], st["news_host"])])
        seq = torch.repeat_interleave(torch.arange(case["B"], device="cuda"),
                                      torch.tensor(st["news_host"], device="cuda"))
        page, within = st["table"].long()[seq, pos // case["page"]], pos % case["page"]
        first = torch.tensor(st["starts_host"][:-1], device="cuda")
        # (64 bits: a value next to the border of two codes goes to the one that it is nearer to)
        k = _rotate(st["k"], pos, case, wide=torch.float64) if case["rot"] else st["k"].double()
        _write_rows(case, st["kc"], st["ks"], k, page, within, page[first], within[first])
        _write_rows(case, st["vc"], st["vs"], st["v"].double(), page, within, page[first], within[first])
        if not case["rot"]:
            return st["kc"], st["vc"], st["ks"], st["vs"]
        st["q_out"].copy_(_rotate(st["q"], pos, case))
        return st["kc"], st["vc"], st["ks"], st["vs"], st["q_out"]
    out = torch.empty_like(st["q"])
    for b, (length, n, t) in enumerate(zip(st["lens_host"], st["news_host"], st["starts_host"])):
        j = torch.arange(length, device="cuda")
        pages = st["table"][b, :-(-length // case["page"])].long()
        k, v = (_values(_pick(c, pages), s[pages]).transpose(0, 1).reshape(case["Hkv"], -1, case["d"])[:, :length]
                for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
        if case["tree"]:
            bits = _tree_bits(st["tree"][t:t + n], n)
            ctx = length - n
            seen = torch.cat((_window(j[:ctx], ctx + bits.sum(dim=1) - 1, case["window"], case["sinks"]), bits), dim=1)
        else:
            seen = _window(j, j[length - n:], case["window"], case["sinks"])
        out[t:t + n] = _attention(st["q"][t:t + n], k, v, seen).to(out.dtype)
    return out


# ----------------------------------------------------------------- work --

def _seen_counts(case, length, n):
    """(query, key) pairs that n new rows of `length` see, and the keys that any of them sees."""
    w, sinks = case["window"], case["sinks"]
    pairs = 0
    for i in range(n):
        pos = length - n + i
        pairs += pos + 1 if not w else min(pos + 1, w + min(sinks, max(0, pos + 1 - w)))
    first = length - n
    union = length if not w else min(length, (length - max(0, first - w + 1)) + min(sinks, max(0, first - w + 1)))
    return pairs, union


def work(case):
    el = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        return {"bytes": case["H"] * case["S"] * case["d"] * el * 2 + 4 * case["S"],
                "flops": 3 * case["H"] * case["S"] * case["rot"]}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        sides, G = 2 if case["glu"] else 1, -(-K // case["group"])
        weight = sides * N * (K // 2 + G * (el + bool(case["zeros"])))
        return {"bytes": weight + M * (K + N * (2 if case["residual"] else 1)) * el, "flops": 2 * sides * M * N * K}
    d, Hkv, H, page = case["d"], case["Hkv"], case["H"], case["page"]
    total = {"bytes": 0, "flops": 0}
    for length, n in zip(*_counts(case)):
        if case["op"] == "append":
            total["bytes"] += n * d * (2 * Hkv * (el + 1) + (2 * H * el if case["rot"] else 0))
            total["bytes"] += 2 * Hkv * (-(-length // page) - (length - n) // page) + 4
            total["flops"] += n * (3 * (H + Hkv) * case["rot"] + 2 * Hkv * d)
        else:
            pairs, union = _seen_counts(case, length, n)
            total["bytes"] += 2 * union * Hkv * d + 2 * n * H * d * el + (4 + 2 * Hkv) * -(-union // page)
            total["flops"] += 4 * d * H * pairs
    return total


# ---------------------------------------------------------------- exact --

def _exact_angles(case):
    """(frequency of every pair, factor): one pair at a time, on the host."""
    rot, kind, s = case["rot"], case.get("scaling", "none"), case.get("factor", 1.0)
    out = []
    for i in range(rot // 2):
        w = math.pow(BASE, -2.0 * i / rot)
        if kind == "linear":
            w /= s
        elif kind == "base" and rot > 2:
            w = math.pow(BASE * math.pow(s, rot / (rot - 2.0)), -2.0 * i / rot)
        elif kind == "bands":
            # Pairs that turn at least 4 times over the original context stay, under one turn are stretched.
            turns = case["original"] * w / (2 * math.pi)
            if turns < 1:
                w /= s
            elif turns < 4:
                part = (turns - 1) / 3
                w = part * w + (1 - part) * w / s
        elif kind == "parts":
            # The pairs that turn 32 times and once bound a ramp over the pairs' numbers.
            at = [rot * math.log(case["original"] / (2 * math.pi * r)) / (2 * math.log(BASE)) for r in (32, 1)]
            a, b = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            part = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            w = (1 - part) * w + part * w / s
        out.append(w)
    return out, (0.1 * math.log(s) + 1 if kind == "parts" else 1.0)


def _exact_rotary(x, pos, case, transpose=False):
    """x [T, heads, d] at positions [T]."""
    out = x.double().clone()
    freqs, m = _exact_angles(case)
    for i, w in enumerate(freqs):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + case["rot"] // 2)
        angle = (pos.double() * w)[:, None]
        c, s = m * torch.cos(angle), m * torch.sin(angle) * (-1 if transpose else 1)
        xa, xb = x[..., a].double(), x[..., b].double()
        out[..., a], out[..., b] = xa * c - xb * s, xa * s + xb * c
    return out


def _exact_codes(x):
    """The e4m3 number that is nearest to x (64 bits), of two as near the one with an even code."""
    numbers = torch.arange(127, dtype=torch.uint8, device=x.device).view(E4M3).double()
    middles = (numbers[1:] + numbers[:-1]) / 2
    code = torch.bucketize(x.abs().contiguous(), middles)  # how many middles lie below
    tie = x.abs() == middles[code.clamp(max=125)]
    return torch.copysign(numbers[torch.where(tie, code + code % 2, code)], x)


def _exact_append(case, codes, scales, rows, table, lens, news, starts):
    """The cache's codes (64 bits) and scale bytes after rows [T, Hkv, d] came, a sequence and a page at a time."""
    codes, scales, page = codes.double(), scales.to(torch.int64), case["page"]
    powers = torch.tensor([2.0 ** k for k in range(-255, 256)], dtype=torch.float64, device=codes.device)
    for b, (length, n, t) in enumerate(zip(lens, news, starts)):
        j = length - n
        while j < length:
            end = min(length, (j // page + 1) * page)
            p, r0, r1 = table[b][j // page], j % page, j % page + end - j
            block = rows[t + j - (length - n):t + end - (length - n)].transpose(0, 1)  # [Hkv, rows, d]
            top = block.abs().amax(dim=(1, 2))
            byte = torch.full_like(scales[p], SCALE_LO)
            for h, value in enumerate(top.tolist()):
                e = SCALE_LO - SCALE_BIAS
                if value > 0:
                    e = max(e, math.frexp(value)[1] - 10)
                    while value > E4M3_MAX * 2.0 ** e and e < SCALE_HI - SCALE_BIAS:
                        e += 1
                byte[h] = e + SCALE_BIAS
            if r0 > 0:
                byte = torch.maximum(byte, scales[p])
                ratio = powers[scales[p] - byte + 255][:, None, None]
                codes[p, :, :r0] = _exact_codes(codes[p, :, :r0] * ratio)
            scales[p] = byte
            factor = powers[byte - SCALE_BIAS + 255][:, None, None]
            codes[p, :, r0:r1] = _exact_codes((block / factor).clamp(-E4M3_MAX, E4M3_MAX))
            j = end
    return codes, scales.to(torch.uint8)


def _exact_attention(q, k, v, allowed):
    """q [n, H, d], k and v [L, Hkv, d] (64 bits), allowed [n, L]; one head at a time."""
    n, H, d = q.shape
    out = torch.zeros(n, H, d, dtype=torch.float64, device=q.device)
    some = allowed.any(dim=1)
    for h in range(H):
        kh, vh = (t[:, h // (H // k.shape[1])].contiguous() for t in (k, v))
        s = (q[:, h].double() @ kh.t().contiguous()) * d ** -0.5
        s[~allowed] = -math.inf
        w = torch.exp(s[some] - s[some].max(dim=1).values[:, None])
        out[some, h] = (w @ vh) / w.sum(dim=1)[:, None]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(st["x"].transpose(0, 1), st["positions"], case, case["grad"]).transpose(0, 1)
    if case["op"] == "linear":
        x, group, sums = st["x"].double(), case["group"], []
        for codes, scales, zeros in zip(st["codes"], st["scales"], st["zeros"]):
            y = torch.zeros(case["M"], case["N"], dtype=torch.float64, device="cuda")
            for g in range(scales.shape[1]):
                part = slice(g * group, min((g + 1) * group, case["K"]))
                levels = codes[:, part].double() - (zeros[:, g:g + 1].double() if zeros is not None else 8)
                y += (x[:, part] @ levels.t().contiguous()) * scales[:, g].double()
            sums.append(y)
        y = sums[0]
        if case["glu"]:
            y = y * torch.sigmoid(y) * sums[1]
        return y if st["residual"] is None else y + st["residual"].double()
    table = st["table"].cpu().tolist()
    if case["op"] == "append":
        seqs = list(zip(st["lens_host"], st["news_host"]))
        pos = torch.tensor([p for length, n in seqs for p in range(length - n, length)], device="cuda")
        k = _exact_rotary(st["k"], pos, case) if case["rot"] else st["k"].double()
        where = (table, st["lens_host"], st["news_host"], st["starts_host"])
        kc, ks = _exact_append(case, st["kc"], st["ks"], k, *where)
        vc, vs = _exact_append(case, st["vc"], st["vs"], st["v"].double(), *where)
        return (kc, vc, ks, vs) + ((_exact_rotary(st["q"], pos, case),) if case["rot"] else ())
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    window = case["window"] or 2 ** 40
    for b, (length, n, t) in enumerate(zip(st["lens_host"], st["news_host"], st["starts_host"])):
        key = torch.arange(length, device="cuda")[None]
        spots = torch.tensor([table[b][j // case["page"]] * case["page"] + j % case["page"] for j in range(length)],
                             device="cuda")
        rows = []
        for codes, scales in ((st["kc"], st["ks"]), (st["vc"], st["vs"])):
            byte = scales[spots // case["page"]].double()
            x = _raw(codes).transpose(1, 2).reshape(-1, case["Hkv"], case["d"])[spots].view(E4M3).double()
            rows.append(x * torch.pow(2.0, byte - SCALE_BIAS)[:, :, None].contiguous())
        ctx = length - n
        if case["tree"]:
            node = torch.zeros(n, n, dtype=torch.bool)
            for i, words in enumerate(st["tree"][t:t + n].cpu().tolist()):
                for w, word in enumerate(words):
                    for bit in range(min(64, n - 64 * w)):
                        node[i, 64 * w + bit] = bool((word >> bit) & 1)
            node = node.cuda()
            at = ctx - 1 + node.sum(dim=1)[:, None]
            allowed = (key < ctx) & ((at - key < window) | (key < case["sinks"]))
            allowed[:, ctx:] = node
        else:
            at = torch.arange(ctx, length, device="cuda")[:, None]
            allowed = (key <= at) & ((at - key < window) | (key < case["sinks"]))
        out[t:t + n] = _exact_attention(st["q"][t:t + n], *rows, allowed)
    return out
