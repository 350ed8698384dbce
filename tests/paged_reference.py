"""The paged cache's operators by their definitions, in 64 bits on the CPU, one
sequence, row and head at a time: what the tests hold the kernels to."""
import numpy as np


def table_rows(table_row, page_size, pages, j):
    """(page, offset) of row j, or None where the table names no page."""
    if j < 0 or j >= len(table_row) * page_size:
        return None
    p = int(table_row[j // page_size])
    return (p, j % page_size) if 0 <= p < pages else None


def sees(i, j, n, length, window, sinks, node_bits=None):
    """Whether new row i of n sees key j of a sequence of `length` rows."""
    if j < 0 or j >= length:
        return False
    pos = length - n + i
    if node_bits is not None:
        ctx = length - n
        if j >= ctx:
            return bool(node_bits[j - ctx])
        pos = ctx - 1 + int(sum(bool(b) for b in node_bits))
    elif j > pos:
        return False
    return not window or j > pos - window or j < sinks


def attention(q, kc, vc, table, lens, starts, window=None, sinks=0, bits=None, scale=None):
    """q [T, H, d], kc and vc [pages, Hkv, page_size, d], bits [T][nodes]; rows of no sequence are NaN."""
    q, kc, vc = (np.asarray(t, np.float64) for t in (q, kc, vc))
    T, H, d = q.shape
    pages, Hkv, page, _ = kc.shape
    scale = 1 / np.sqrt(d) if scale is None else scale
    out = np.full((T, H, d), np.nan)
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        spots = [(j, table_rows(table[b], page, pages, j)) for j in range(length)]
        spots = [(j, s) for j, s in spots if s is not None]
        for i in range(n):
            t = starts[b] + i
            seen = [s for j, s in spots if sees(i, j, n, length, window, sinks, None if bits is None else bits[t])]
            if not seen:
                out[t] = 0
                continue
            P, O = np.array(seen).T
            for h in range(H):
                kv = h // (H // Hkv)
                s = kc[P, kv, O] @ q[t, h] * scale
                w = np.exp(s - s.max())
                out[t, h] = w @ vc[P, kv, O] / w.sum()
    return out


def tree_bits(parents):
    """Node i's ancestors and itself, for parents below their nodes (else a root)."""
    rows = []
    for i, p in enumerate(parents):
        r = list(rows[p]) + [0] * (len(parents) - len(rows[p])) if 0 <= p < i else [0] * len(parents)
        r[i] = 1
        rows.append(r)
    return rows


def rope(x, pos, base):
    """x [..., d] rotated by position pos."""
    x = np.asarray(x, np.float64)
    half = x.shape[-1] // 2
    a = pos * base ** (-np.arange(half) / half)
    x1, x2 = x[..., :half], x[..., half:]
    return np.concatenate((x1 * np.cos(a) - x2 * np.sin(a), x2 * np.cos(a) + x1 * np.sin(a)), axis=-1)
