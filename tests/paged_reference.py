"""Plain 64-bit forms of the paged-cache operators and of the token draw, for their tests."""
import numpy as np

import oracle_lib as O


def value(codes):
    """The real numbers that xlns16 codes stand for, as the attention reads them (up to the largest half)."""
    c = np.asarray(codes).astype(np.int64) & 0xffff
    log = np.minimum(c & 0x7fff, 0x47ff)
    v = np.where(log == 0, 0.0, np.exp2((log - 0x4000) / 128.0))
    return np.where(c & 0x8000, -v, v)


class Cache:
    """Pages on the host: k, v int16 [n_pages, n_head_kv, page * head_dim], filled with `fill`."""

    def __init__(self, n_pages, page, nkv, hd, fill=0x47ff):
        self.page, self.nkv, self.hd, self.n_pages = page, nkv, hd, n_pages
        self.k = np.full((n_pages, nkv, page * hd), fill, np.uint16)
        self.v = self.k.copy()

    def at(self, p, d):
        """Offsets of (cell p of a page, dim d) in a head's keys and values."""
        return ((d // 8) * self.page + p) * 8 + d % 8, ((p // 8) * self.hd + d) * 8 + p % 8

    def put(self, table_row, cells, k, v):
        """Codes k, v [len(cells), nkv, hd] into the cells of a sequence."""
        d = np.arange(self.hd)
        for i, c in enumerate(cells):
            pg = table_row[c // self.page]
            ko, vo = self.at(c % self.page, d)
            self.k[pg][:, ko] = k[i]
            self.v[pg][:, vo] = v[i]

    def get(self, table_row, n):
        """Codes [n, nkv, hd] of a sequence's first n cells."""
        c = np.arange(n)
        pg = np.asarray(table_row)[c // self.page]
        ko, vo = self.at(c[:, None] % self.page, np.arange(self.hd)[None])
        return (self.k[pg][np.arange(n)[:, None, None], np.arange(self.nkv)[None, :, None], ko[:, None]],
                self.v[pg][np.arange(n)[:, None, None], np.arange(self.nkv)[None, :, None], vo[:, None]])


def tables(rng, kv_len, page, width=None, spare=2):
    """A table with the sequences' pages in random order (-1 past them), and the pages in all."""
    need = [max(0, -(-int(n) // page)) for n in kv_len]
    n_pages = sum(need) + spare
    order = rng.permutation(n_pages)
    t = np.full((len(need), width or max(need + [1])), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, n_pages


def attention(q, keys, vals, pos, scale, window=0, hidden=()):
    """One sequence: q [T, nh, hd] float32, keys / vals [n, nkv, hd] codes, pos [T].  Returns the
    outputs in 64 bits and a bound of the error of each (see tolerance())."""
    T, nh, hd = q.shape
    n, nkv = keys.shape[:2]
    K, V = value(keys), value(vals)
    out, tol = np.zeros((T, nh, hd)), np.zeros((T, nh, hd))
    for t in range(T):
        lo = max(0, pos[t] - window + 1) if window else 0
        j = np.array([c for c in range(lo, min(pos[t] + 1, n)) if c not in hidden], dtype=int)
        if len(j) == 0:
            continue
        for h in range(nh):
            g = h // (nh // nkv)
            qd = q[t, h].astype(np.float64)
            s = scale * (K[j, g] @ qd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ V[j, g]
            tol[t, h] = tolerance(np.abs(scale) * (np.abs(K[j, g]) @ np.abs(qd)).max(), np.abs(qd).sum() * abs(scale),
                                  p, V[j, g], hd)
    return out, tol


def tolerance(A, Q, p, V, hd):
    """A bound of the attention's error.  Scores: each operand is a pair of halves, off by 2^-22 of
    itself (2^-36 where a key is below the normal halves), the product of the two low halves is left
    out (2^-22), the decoding power is off by one step (2^-23), and hd terms are summed in 32 bits
    (hd 2^-24, twice: the high and the cross products).  With A the largest sum of the products'
    magnitudes a score is off by d, so its weight by a factor within 1 +- (d + 2^-22), numerator and
    denominator alike; the weights are halves in pairs too, the values as the keys, and n terms are
    summed in 32 bits (n 2^-24, twice).  (The weights' own floor: 2^-39.)"""
    n = len(p)
    d = A * (4 * 2.0 ** -22 + hd * 2.0 ** -23) + Q * 2.0 ** -36
    rel = 2 * (d + 2.0 ** -22) + 5 * 2.0 ** -22 + n * 2.0 ** -22
    return rel * (p @ np.abs(V)) + n * (2.0 ** -36) + 2.0 ** -38 * np.abs(V).sum(0)


def rope(x, cs, neox, nd):
    """x [T, heads, hd] float32 rotated in xlns16 (its first nd dims, cs [T, nd / 2, 2]): the F32 values."""
    L = O.lib()
    c = O.f2x16(np.ascontiguousarray(x))
    out = c.copy()
    cc, ss = O.f2x16(np.ascontiguousarray(cs[..., 0])), O.f2x16(np.ascontiguousarray(cs[..., 1]))
    half = nd // 2
    for t in range(x.shape[0]):
        for h in range(x.shape[1]):
            for j in range(half):
                i0, i1 = (j, j + half) if neox else (2 * j, 2 * j + 1)
                a, b, co, si = int(c[t, h, i0]), int(c[t, h, i1]), int(cc[t, j]), int(ss[t, j])
                out[t, h, i0] = L.lno16_add(L.lno16_mul(a, co), L.lno16_mul(b, si) ^ 0x8000)
                out[t, h, i1] = L.lno16_add(L.lno16_mul(a, si), L.lno16_mul(b, co))
    return O.x2f16(out)


def store_codes(x):
    """The cache codes of F32 values: through IEEE half."""
    with np.errstate(over="ignore"):
        return O.f2x16(np.ascontiguousarray(x.astype(np.float16).astype(np.float32)))


def kept(row, T, top_k, top_p, min_p):
    """The kept tokens of a row by rank, and their weights in 64 bits."""
    x = row.astype(np.float64)
    ok = np.nonzero(x > -np.inf)[0]
    order = ok[np.argsort(-x[ok], kind="stable")]
    if len(order) == 0:
        return order, np.zeros(0)
    d = np.where(x[order] == x[order[0]], 0.0, x[order] - x[order[0]])
    w = np.exp(d / T)
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    n = len(w)
    if top_p < 1:
        c = np.cumsum(w)
        n = min(n, 1 + int(np.searchsorted(c, top_p * c[-1], side="left")))
    if min_p > 0:
        n = min(n, max(1, int((w >= min_p).sum())))
    return order[:n], w[:n]


def draw(row, T, top_k, top_p, min_p, u):
    """(token, probability, the distance of u from the nearest border of the token's share)."""
    x = np.asarray(row)
    with np.errstate(invalid="ignore"):
        if not (x > -np.inf).any():
            return -1, 0.0, 1.0
        if not T > 0:
            return int(np.nanargmax(np.where(np.isnan(x), -np.inf, x))), 1.0, 1.0
        order, w = kept(x, T, top_k, top_p, min_p)
    idx = np.argsort(order)
    tok, w = order[idx], w[idx]
    c = np.cumsum(w) / w.sum()
    at = int(np.searchsorted(c, min(max(u, 0.0), 1 - 1e-12), side="right"))
    at = min(at, len(c) - 1)
    return int(tok[at]), w[at] / w.sum(), float(np.abs(c[:-1] - u).min()) if len(c) > 1 else 1.0
