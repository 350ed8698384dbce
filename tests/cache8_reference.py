"""The 8-bit paged cache by its definition, in 64 bits on the CPU: what the tests
hold the kernels to.  A cache is (codes [pages, Hkv, page_size, d] and scales
[pages, Hkv], uint8 arrays), K's or V's."""
import numpy as np

from paged_reference import table_rows

LO, HI = 17, 246


def numbers():
    """The value of every code (index), codes 127 and 255 NaN."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7), f * 2.0 ** -9)
    v[(c & 127) == 127] = np.nan
    return np.where(c & 128, -v, v)


NUM = numbers()
POS = NUM[:127]
MID = (POS[1:] + POS[:-1]) / 2


def encode(x):
    """The nearest codes of x (64 bits), of two as near the even one; beyond 448 saturated, infinities and NaN as NaN."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    c = np.searchsorted(MID, a)
    tie = a == MID[np.minimum(c, 125)]
    c = np.where(tie & (c % 2 == 1), c + 1, c)
    c = np.where(np.isfinite(a), np.minimum(c, 126), 127)
    return (c | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_of(top):
    """The smallest exponent byte that holds magnitude `top`."""
    s = LO
    while s < HI and top > 448 * 2.0 ** (s - 127):
        s += 1
    return s


def values(codes, scales):
    return NUM[codes] * 2.0 ** (scales.astype(np.float64) - 127)[:, :, None, None]


def same(a, b):
    """Equal codes, zeros of either sign and NaN of either sign being equal."""
    return ((a == b) | ((a & 127 == 0) & (b & 127 == 0)) | ((a & 127 == 127) & (b & 127 == 127)))


def append(codes, scales, rows, table, lens, starts, max_q=None):
    """New rows [T, Hkv, d] (64 bits) into copies of the cache."""
    codes, scales = codes.copy(), scales.copy()
    pages, Hkv, size, d = codes.shape
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        use = n if max_q is None else min(n, max_q)
        spots = [(i, table_rows(table[b], size, pages, length - n + i)) for i in range(use)]
        by_page = {}
        for i, s in spots:
            if s is not None:
                by_page.setdefault(s[0], []).append((i, s[1]))
        for p, entries in by_page.items():
            first = entries[0][1]
            for h in range(Hkv):
                block = np.array([rows[starts[b] + i, h] for i, _ in entries])
                a = np.abs(block)
                s = scale_of(a[np.isfinite(a)].max(initial=0))
                if first > 0:
                    old = int(scales[p, h])
                    s = max(s, old)
                    if s > old:
                        codes[p, h, :first] = encode(NUM[codes[p, h, :first]] * 2.0 ** (old - s))
                scales[p, h] = s
                for (_, o), row in zip(entries, block):
                    codes[p, h, o] = encode(row * 2.0 ** (127 - s))
    return codes, scales


def accept(codes, scales, table, lens, news, paths):
    """The accepted paths kept, in copies of the cache of one layer."""
    codes, scales = codes.copy(), scales.copy()
    old_codes, old_scales = codes.copy(), scales.copy()
    pages, Hkv, size, d = codes.shape
    for b, (length, n, path) in enumerate(zip(lens, news, paths)):
        ctx = length - n
        moves = [(table_rows(table[b], size, pages, ctx + i), table_rows(table[b], size, pages, ctx + node), i)
                 for i, node in enumerate(path) if i != node]
        by_page = {}
        for dst, src, i in moves:
            if dst is not None and src is not None:
                by_page.setdefault(dst[0], []).append((dst[1], src))
        first_row = ctx + next((i for i, node in enumerate(path) if i != node), len(path))
        for p, entries in by_page.items():
            kept = first_row % size if table_rows(table[b], size, pages, first_row)[0] == p else 0
            for h in range(Hkv):
                s = max([int(old_scales[src[0], h]) for _, src in entries] + ([int(old_scales[p, h])] if kept else []))
                shift = lambda row, at: encode(NUM[row] * 2.0 ** (int(old_scales[at, h]) - s))  # noqa: E731
                if kept and s > old_scales[p, h]:
                    codes[p, h, :kept] = shift(old_codes[p, h, :kept], p)
                for o, src in entries:
                    codes[p, h, o] = shift(old_codes[src[0], h, src[1]], src[0])
                scales[p, h] = s
    return codes, scales


def rotate(x, pos, r):
    """x [T, heads, d] (64 bits) at positions [T] by an ops.Rotary."""
    y = np.array(x, np.float64)
    for i, f in enumerate(r.frequencies):
        a, b = (2 * i, 2 * i + 1) if r.interleaved else (i, i + r.dim // 2)
        t = (np.asarray(pos, np.float64) * f)[:, None]
        c, s = r.gain * np.cos(t), r.gain * np.sin(t)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def rotate_bound(x, want, r, finfo):
    """How far rows rotated in fp32 may be off: sine, cosine, their products and the sum are rounded by 2^-24 of at
    most gain (|x1| + |x2|), three times over, and the result by half a step of its type."""
    pair = np.zeros(x.shape)
    half = r.dim // 2
    a, b = (slice(0, r.dim, 2), slice(1, r.dim, 2)) if r.interleaved else (slice(0, half), slice(half, r.dim))
    pair[..., a] = pair[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    inner = (3 * 2.0 ** -24 + 2.0 ** -30) * abs(r.gain) * pair
    return inner + finfo.eps / 2 * (np.abs(want) + inner) + finfo.tiny * finfo.eps / 2
