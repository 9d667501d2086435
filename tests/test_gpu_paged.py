"""The paged xlns16 cache on the GPU: stores bit for bit against the oracle and the contiguous
cache's operators, attention against a 64-bit form within a bound derived from its arithmetic
(paged_reference.tolerance), lengths from one token on, odd sizes, windows, empty rows, bad pages,
rows of no sequence, other strides, streams and captured graphs."""
import numpy as np
import pytest

import oracle_lib as O
import paged_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ln():
    import lnship
    import lnship.paged
    lnship.init()
    return lnship


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def starts(q_len, first=0):
    return (first + np.concatenate([[0], np.cumsum(q_len)])).astype(np.int32)


def positions(q_len, kv_len):
    return [np.arange(m - n, m) for n, m in zip(q_len, kv_len)]


def rope_table(ln, n_pos, nd, theta=10000.0):
    import ctypes
    t = np.empty((n_pos, nd // 2, 2), np.float32)
    ln.check(ln.lib().lnship_rope_table(theta, nd, n_pos, ctypes.c_void_p(t.ctypes.data)))
    return t


# ---- stores ------------------------------------------------------------------------

STORES = [
    # q_len, kv_len, page, heads, kv heads, dim, rotated, neox
    ([1], [1], 16, 1, 1, 8, 8, False),
    ([1], [301], 16, 9, 3, 64, 64, False),
    ([1, 1, 1], [17, 64, 5], 32, 8, 2, 128, 128, True),
    ([19, 1, 40], [19, 77, 53], 16, 4, 2, 64, 64, True),
    ([33, 0, 7], [50, 9, 7], 64, 3, 1, 80, 80, False),
    ([9, 12], [9, 30], 16, 2, 2, 40, 20, True),
    ([9, 12], [25, 12], 16, 2, 2, 72, 18, False),
    ([5], [261], 256, 6, 6, 256, 64, True),
    ([21], [23], 16, 5, 5, 24, 0, False),
    # 2^19 values and more: tables in LDS, a row or eight to a workgroup
    ([300, 1, 40], [310, 9, 47], 16, 24, 8, 64, 64, False),
    ([1] * 90, list(range(1, 91)), 64, 32, 8, 128, 128, True),
    ([700, 350], [700, 401], 32, 4, 2, 80, 80, True),
    ([1100], [1117], 16, 2, 2, 96, 48, False),
    ([1030, 0, 3], [1030, 5, 3], 256, 3, 1, 128, 64, True),
    ([8200], [8200], 64, 3, 2, 8, 8, False),
]


@pytest.mark.parametrize("q_len,kv_len,page,nh,nkv,hd,nd,neox", STORES)
@pytest.mark.parametrize("fused", [True, False])
def test_stores_equal_the_oracle(ln, q_len, kv_len, page, nh, nkv, hd, nd, neox, fused):
    print(f"\n[store] {q_len} {kv_len} page {page} {nh}/{nkv}x{hd} rot {nd} neox {neox} fused {fused}", flush=True)
    rng = np.random.default_rng(hd * 7 + nh)
    T = sum(q_len)
    x = (rng.standard_normal((T, nh + 2 * nkv, hd)) * 3).astype(np.float32)
    x[0, :, :4] = [0.0, -0.0, 1e-30, 7e4]          # zeros, an underflow and an overflow of the half
    table, n_pages = R.tables(rng, kv_len, page)
    c = R.Cache(n_pages, page, nkv, hd, fill=0x1234)
    k, v = dev(c.k), dev(c.v)
    cs = rope_table(ln, max(kv_len), nd) if nd else None
    pos = np.concatenate(positions(q_len, kv_len))
    if fused:
        xd = dev(x)
        q_, k_, v_ = xd[:, :nh], xd[:, nh:nh + nkv], xd[:, nh + nkv:]
    else:
        q_, k_, v_ = dev(x[:, :nh]), dev(x[:, nh:nh + nkv]), dev(x[:, nh + nkv:])
    out = ln.paged.rope_store_kv(q_, k_, v_, k, v, page, dev(table), dev(starts(q_len)), dev(np.int32(kv_len)),
                                 dev(cs) if nd else None, n_dims=nd, neox=neox)
    rot = R.rope(x[:, :nh + nkv], cs[pos], neox, nd) if nd else x[:, :nh + nkv]
    kc, vc = R.store_codes(rot[:, nh:]), R.store_codes(x[:, nh + nkv:])
    at = 0
    for s, p in enumerate(positions(q_len, kv_len)):
        c.put(table[s], p, kc[at:at + len(p)], vc[at:at + len(p)])
        at += len(p)
    assert np.array_equal(k.cpu().numpy().view(np.uint16), c.k)     # other cells untouched
    assert np.array_equal(v.cpu().numpy().view(np.uint16), c.v)
    assert np.array_equal(out.cpu().numpy().view(np.uint32), rot[:, :nh].view(np.uint32))


def test_stores_equal_the_contiguous_caches(ln):
    """The codes and queries of lnship16_rope_store_kv for the same tokens."""
    import ctypes
    rng = np.random.default_rng(3)
    nh, nkv, hd, page, n = 9, 3, 64, 16, 45
    x = rng.standard_normal((n, nh + 2 * nkv, hd)).astype(np.float32)
    cs = dev(rope_table(ln, 64, hd))
    xd = dev(x)
    kc = torch.zeros(nkv * hd * 64, dtype=torch.int16, device="cuda")
    vc = torch.zeros_like(kc)
    q = torch.empty((n, nh, hd), device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    P = lambda t: ctypes.c_void_p(t.data_ptr())
    a = ln.QkvStoreArgs(P(xd), (nh + 2 * nkv) * hd, P(pos), n, nh, nkv, hd, hd, P(cs), P(q), P(kc), P(vc), 64, hd * 64,
                        hd * 64, None, 0)
    ln.check(ln.lib().lnship16_rope_store_kv(ctypes.byref(a), ln._stream()))
    table, n_pages = R.tables(rng, [n], page)
    k, v = ln.paged.alloc_pages(n_pages, page, nkv, hd)
    q2 = ln.paged.rope_store_kv(xd[:, :nh], xd[:, nh:nh + nkv], xd[:, nh + nkv:], k, v, page, dev(table),
                                dev(np.int32([0, n])), dev(np.int32([n])), cs)
    assert torch.equal(q, q2)
    c = R.Cache(n_pages, page, nkv, hd)
    c.k, c.v = k.cpu().numpy().view(np.uint16), v.cpu().numpy().view(np.uint16)
    keys, vals = c.get(table[0], n)
    d = np.arange(hd)
    ref_k = kc.cpu().numpy().view(np.uint16).reshape(nkv, -1)
    ref_v = vc.cpu().numpy().view(np.uint16).reshape(nkv, -1)
    for p in range(n):
        assert np.array_equal(keys[p], ref_k[:, ((d // 8) * 64 + p) * 8 + d % 8])
        assert np.array_equal(vals[p], ref_v[:, ((p // 8) * hd + d) * 8 + p % 8])


@pytest.mark.parametrize("ld_extra,shift", [(0, 0), (1, 0), (4, 1), (8, 0)])
def test_store_strides_and_rows_of_no_sequence(ln, ld_extra, shift):
    """Rows of other strides and alignments; rows before the first and behind the last sequence."""
    rng = np.random.default_rng(5)
    nh, nkv, hd, page = 2, 1, 32, 16
    q_len, kv_len, T = [3, 10], [3, 21], 17       # rows 2 .. 14
    start = starts(q_len, first=2)
    cs = rope_table(ln, 32, hd)
    ld = nh * hd + ld_extra
    buf = rng.standard_normal(T * ld + 8).astype(np.float32)
    q = torch.as_strided(dev(buf), (T, nh, hd), (ld, hd, 1), shift)
    kv = rng.standard_normal((T, 2, hd)).astype(np.float32)
    table, n_pages = R.tables(rng, kv_len, page)
    k, v = ln.paged.alloc_pages(n_pages, page, nkv, hd)
    kd = dev(kv)
    out = torch.full((T, nh, hd), 7.0, device="cuda")
    ln.paged.rope_store_kv(q, kd[:, :1], kd[:, 1:], k, v, page, dev(table), dev(start), dev(np.int32(kv_len)), dev(cs),
                           out=out)
    c = R.Cache(n_pages, page, nkv, hd, fill=0)
    pos = positions(q_len, kv_len)
    rot_q = R.rope(q.cpu().numpy()[2:15], cs[np.concatenate(pos)], False, hd)
    rot_k = R.rope(kv[2:15, :1], cs[np.concatenate(pos)], False, hd)
    kc, vc = R.store_codes(rot_k), R.store_codes(kv[2:15, 1:])
    c.put(table[0], pos[0], kc[:3], vc[:3])
    c.put(table[1], pos[1], kc[3:], vc[3:])
    o = out.cpu().numpy()
    assert np.array_equal(o[2:15], rot_q)
    assert (o[:2] == 7.0).all() and (o[15:] == 7.0).all()
    assert np.array_equal(k.cpu().numpy().view(np.uint16), c.k) and np.array_equal(v.cpu().numpy().view(np.uint16), c.v)


@pytest.mark.parametrize("T,nh,nkv,hd", [(150, 24, 16, 64), (1200, 4, 2, 64)])
def test_stores_of_many_rows_strided_with_bad_pages(ln, T, nh, nkv, hd):
    """Rows before the first and behind the last sequence, a bad page, positions past the rope table."""
    rng = np.random.default_rng(T)
    page, first = 16, 5
    q_len = [T - 60, 40]
    kv_len = [T - 60 + 3, 40]
    n_pos = T - 62                    # the last five of the first sequence lie behind it
    table, n_pages = R.tables(rng, kv_len, page)
    start = starts(q_len, first)
    cs = rope_table(ln, T, hd)
    ld = nh * hd + 4
    q = torch.as_strided(dev(rng.standard_normal(T * ld).astype(np.float32)), (T, nh, hd), (ld, hd, 1), 0)
    kv = dev((rng.standard_normal((T, 2, nkv, hd)) * 2).astype(np.float32))
    k, v = ln.paged.alloc_pages(n_pages, page, nkv, hd)
    bad = table.copy()
    bad[1, 1] = n_pages + 7           # cells 16 .. 31 of the second sequence
    index_error(ln)
    out = torch.full((T, nh, hd), 7.0, device="cuda")
    ln.paged.rope_store_kv(q, kv[:, 0], kv[:, 1], k, v, page, dev(bad), dev(start), dev(np.int32(kv_len)), dev(cs[:n_pos]),
                           out=out)
    assert index_error(ln)[0] == 1
    pos = positions(q_len, kv_len)
    rows = np.arange(first, first + T - 20)
    p, s = np.concatenate(pos), np.repeat([0, 1], q_len)
    ok = p < n_pos
    x, kvn = q.cpu().numpy(), kv.cpu().numpy()
    rot = R.rope(np.concatenate([x[rows], kvn[rows, 0]], 1), cs[p], False, hd)
    o = out.cpu().numpy()
    assert np.array_equal(o[rows[ok]], rot[ok][:, :nh])
    rest = np.setdiff1d(np.arange(T), rows[ok])
    assert len(rest) == 25 and (o[rest] == 7.0).all()
    kc, vc = R.store_codes(rot[:, nh:]), R.store_codes(kvn[rows, 1])
    c = R.Cache(n_pages, page, nkv, hd, fill=0)
    for i in (0, 1):
        m = ok & (s == i) & ~((s == 1) & (p // page == 1))
        c.put(table[i], p[m], kc[m], vc[m])
    assert np.array_equal(k.cpu().numpy().view(np.uint16), c.k) and np.array_equal(v.cpu().numpy().view(np.uint16), c.v)


def index_error(ln):
    import ctypes
    bad = ctypes.c_int64(0)
    return ln.lib().lnship_index_error(ctypes.byref(bad), ln._stream()), bad.value


@pytest.mark.parametrize("what", ["negative position", "past the table", "past the rope table", "bad page"])
def test_bad_positions_and_pages_are_recorded(ln, what):
    """Recorded and skipped: the other rows are stored, nothing else is written."""
    print(f"\n[store] {what}", flush=True)
    rng = np.random.default_rng(6)
    nh, nkv, hd, page = 2, 1, 16, 16
    q_len, kv_len, n_pos = [4, 3], [4, 20], 64
    table, n_pages = R.tables(rng, kv_len, page)
    good = {0, 1, 2, 3}
    want = {"negative position": -2, "past the table": 32, "past the rope table": 18, "bad page": 1000}[what]
    if what == "negative position":
        kv_len[1] = 1            # positions -2, -1, 0
        good |= {6}
    elif what == "past the table":
        kv_len[1] = 35           # positions 32 .. 34; the table holds 32
    elif what == "past the rope table":
        n_pos = 18               # positions 17, 18, 19
        good |= {4}
    else:
        table[1, 1] = 1000
    index_error(ln)
    x = rng.standard_normal((7, nh + 2 * nkv, hd)).astype(np.float32)
    xd, cs = dev(x), rope_table(ln, 64, hd)
    k, v = ln.paged.alloc_pages(n_pages, page, nkv, hd)
    out = torch.full((7, nh, hd), 7.0, device="cuda")
    ln.paged.rope_store_kv(xd[:, :nh], xd[:, nh:nh + 1], xd[:, nh + 1:], k, v, page, dev(table), dev(starts(q_len)),
                           dev(np.int32(kv_len)), dev(cs[:n_pos]), out=out)
    found, at = index_error(ln)
    assert found == 1 and (at == want or (what != "bad page" and want <= at <= want + 2))
    assert index_error(ln)[0] == 0
    c = R.Cache(n_pages, page, nkv, hd, fill=0)
    pos = np.concatenate(positions(q_len, kv_len))
    rows = sorted(good)
    rot = R.rope(x[rows][:, :nh + 1], cs[pos[rows]], False, hd)
    for i, r in enumerate(rows):
        c.put(table[0 if r < 4 else 1], [pos[r]], R.store_codes(rot[i:i + 1, nh:]), R.store_codes(x[r:r + 1, nh + 1:]))
    assert np.array_equal(k.cpu().numpy().view(np.uint16), c.k) and np.array_equal(v.cpu().numpy().view(np.uint16), c.v)
    o = out.cpu().numpy()
    assert np.array_equal(o[rows], rot[:, :nh])
    if what != "bad page":       # there the query is in order, only its cell is not
        assert (o[[r for r in range(7) if r not in good]] == 7.0).all()


@pytest.mark.parametrize("T,nh,nkv,hd", [(5, 2, 1, 64), (150, 24, 16, 64)])
def test_a_rope_table_without_positions(ln, T, nh, nkv, hd):
    """Every row is recorded and skipped."""
    k, v = ln.paged.alloc_pages(20, 16, nkv, hd)
    x = torch.ones((T, nh + 2 * nkv, hd), device="cuda")
    cs = torch.ones((1, hd // 2, 2), device="cuda")
    table = dev(np.arange(20, dtype=np.int32)[None])
    out = torch.full((T, nh, hd), 7.0, device="cuda")
    index_error(ln)
    ln.paged.rope_store_kv(x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:], k, v, 16, table, dev(np.int32([0, T])),
                           dev(np.int32([T])), cs[:0], out=out)
    assert index_error(ln)[0] == 1
    assert (out == 7.0).all() and not k.any() and not v.any()


def test_overlapping_rows_are_refused(ln):
    k, v = ln.paged.alloc_pages(2, 16, 1, 32)
    batch = (dev(np.int32([[0, 1]])), dev(np.int32([0, 3])), dev(np.int32([3])))
    one = torch.zeros((1, 2, 32), device="cuda")
    x = torch.zeros((3, 2, 32), device="cuda")
    for q, out in ((one.expand(3, 2, 32), x), (x, torch.zeros((1, 2, 32), device="cuda").expand(3, 2, 32))):
        with pytest.raises(ln.LnshipError, match="overlap"):
            ln.paged.attention(q, k, v, 16, *batch, 1.0, out=out)
        with pytest.raises(ln.LnshipError, match="overlap"):
            ln.paged.rope_store_kv(q, x[:, :1], x[:, 1:], k, v, 16, *batch, None, n_dims=0, out=out)


# ---- attention ------------------------------------------------------------------------

ATTN = [
    # q_len, kv_len, page, heads, kv heads, dim, window
    ([1], [1], 16, 1, 1, 8, 0),
    ([1], [301], 16, 9, 3, 64, 0),
    ([1], [2500], 64, 32, 8, 128, 0),
    ([1, 1, 1, 1], [5, 700, 1, 64], 32, 8, 2, 128, 0),
    ([3, 1, 17], [3, 40, 100], 16, 4, 2, 64, 0),
    ([33, 0, 7, 50], [50, 9, 7, 120], 16, 9, 3, 80, 0),
    ([40], [47], 64, 28, 4, 80, 0),
    ([70, 5], [70, 333], 32, 5, 1, 96, 0),
    ([131], [260], 16, 16, 1, 128, 0),
    ([9], [400], 256, 3, 3, 256, 0),
    ([30], [90], 128, 2, 2, 200, 0),
    ([50], [300], 16, 4, 4, 40, 16),
    ([64, 3], [200, 777], 32, 8, 2, 64, 100),
    ([1], [1000], 16, 12, 4, 64, 33),
    ([257], [257], 64, 8, 2, 128, 129),
    ([300], [300], 16, 9, 3, 64, 0),
    ([520, 1, 90], [800, 50, 90], 32, 8, 2, 64, 0),
    # more workgroups than CUs: four waves each
    ([1] * 40, [1 + 37 * i for i in range(40)], 16, 32, 8, 64, 0),
    ([1] * 40, [1 + 31 * i for i in range(40)], 64, 8, 8, 72, 0),
    ([1] * 40, [2 + 29 * i for i in range(40)], 32, 16, 8, 128, 300),
]


def attn_case(rng, q_len, kv_len, page, nh, nkv, hd, qscale=2.0, kstd=1.0, vstd=1.0, width=None):
    T = sum(q_len)
    table, n_pages = R.tables(rng, kv_len, page, width)
    c = R.Cache(n_pages, page, nkv, hd, fill=0x7fff)     # what lies past the cells: the largest code
    c.v[:, :, ::2] = 0xffff
    keys, vals = [], []
    for s, n in enumerate(kv_len):
        n = max(0, n)
        keys.append(R.store_codes((rng.standard_normal((n, nkv, hd)) * kstd).astype(np.float32)))
        vals.append(R.store_codes((rng.standard_normal((n, nkv, hd)) * vstd).astype(np.float32)))
        c.put(table[s], np.arange(n), keys[-1], vals[-1])
    q = (rng.standard_normal((T, nh, hd)) * qscale).astype(np.float32)
    return q, c, table, keys, vals


def widen(table, page, cells):
    """The same pages in a table of so many cells: what a call costs at most, and by it which kernel runs."""
    wide = np.full((table.shape[0], max(cells // page, table.shape[1])), -1, np.int32)
    wide[:, :table.shape[1]] = table
    return wide


def run_attn(ln, q, c, table, q_len, kv_len, window=0, scale=None, out=None, cells=0):
    table = widen(table, c.page, cells)
    return ln.paged.attention(dev(q), dev(c.k), dev(c.v), c.page, dev(table), dev(starts(q_len)), dev(np.int32(kv_len)),
                              scale if scale is not None else q.shape[2] ** -0.5, window=window, out=out)


def check_attn(got, q, q_len, kv_len, keys, vals, window=0, scale=None, hidden=()):
    at = 0
    scale = scale if scale is not None else q.shape[2] ** -0.5
    for s, p in enumerate(positions(q_len, kv_len)):
        n = len(p)
        ref, tol = R.attention(q[at:at + n], keys[s], vals[s], p, scale, window, hidden)
        err = np.abs(got[at:at + n] - ref)
        bad = ~(err <= tol)
        assert not bad.any(), (s, int(bad.sum()), float(np.nanmax(err / np.maximum(tol, 1e-300))),
                               np.argwhere(bad)[:3].tolist())
        at += n


@pytest.mark.parametrize("q_len,kv_len,page,nh,nkv,hd,window", ATTN)
def test_attention_against_64_bits(ln, q_len, kv_len, page, nh, nkv, hd, window):
    print(f"\n[attn] {q_len} {kv_len} page {page} {nh}/{nkv}x{hd} window {window}", flush=True)
    rng = np.random.default_rng(nh * 1000 + hd)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, page, nh, nkv, hd)
    got = run_attn(ln, q, c, table, q_len, kv_len, window).cpu().numpy()
    check_attn(got, q, q_len, kv_len, keys, vals, window)
    assert np.array_equal(got, run_attn(ln, q, c, table, q_len, kv_len, window).cpu().numpy())   # run to run


@pytest.mark.parametrize("q_len,kv_len,page,nh,nkv,hd,window", [
    ([300], [300], 16, 9, 3, 64, 0), ([70, 5], [70, 333], 32, 5, 1, 96, 0), ([131], [260], 64, 16, 1, 128, 0),
    ([40, 90], [300, 90], 16, 4, 4, 24, 50), ([520, 1, 90], [800, 50, 90], 32, 8, 2, 64, 0)])
def test_chunks_behind_a_table_of_many_pages(ln, q_len, kv_len, page, nh, nkv, hd, window):
    """Tables of more cells than the workspace holds decoded: each workgroup decodes what it sees."""
    rng = np.random.default_rng(hd)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, page, nh, nkv, hd)
    narrow = run_attn(ln, q, c, table, q_len, kv_len, window).cpu().numpy()
    wide = np.full((len(q_len), (1 << 30) // (nkv * 8 * ((hd + 31) // 32 * 32) * page * len(q_len)) + 3), -1, np.int32)
    wide[:, :table.shape[1]] = table
    got = run_attn(ln, q, c, wide, q_len, kv_len, window).cpu().numpy()
    check_attn(got, q, q_len, kv_len, keys, vals, window)
    check_attn(narrow, q, q_len, kv_len, keys, vals, window)


@pytest.mark.parametrize("q_len,kv_len,page,nh,nkv,hd,window", [
    # 64 to 511 rows a sequence: each workgroup decodes; more: decoded before
    ([300], [300], 16, 9, 3, 64, 0), ([70, 5], [70, 333], 32, 5, 1, 96, 0), ([131], [260], 16, 16, 1, 128, 0),
    ([40, 90], [300, 90], 16, 4, 4, 24, 50), ([520, 1, 90], [800, 50, 90], 32, 8, 2, 64, 0), ([65], [65], 256, 2, 2, 8, 0),
    ([600], [900], 16, 1, 1, 32, 0), ([130, 3], [170, 9], 64, 18, 2, 128, 0), ([257], [300], 16, 28, 4, 80, 0),
    ([300, 1, 0, 180], [310, 5, 7, 900], 128, 32, 4, 96, 0), ([520], [530], 64, 8, 2, 128, 129), ([333], [999], 32, 3, 1, 64, 31),
    ([65, 120], [66, 300], 16, 16, 8, 128, 0), ([64, 90, 130], [64, 900, 131], 32, 8, 2, 96, 77), ([75], [333], 64, 4, 1, 112, 0),
    ([1030], [1050], 16, 4, 2, 72, 0), ([519], [700], 32, 8, 2, 104, 0), ([2050], [2050], 64, 2, 2, 128, 700)])
def test_chunks_behind_wide_tables(ln, q_len, kv_len, page, nh, nkv, hd, window):
    print(f"\n[attn] {q_len} {kv_len} page {page} {nh}/{nkv}x{hd} window {window}, wide", flush=True)
    rng = np.random.default_rng(nh * 1000 + hd)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, page, nh, nkv, hd)
    cells = (1 << 28) // (sum(q_len) * nh * hd) + 2 * page
    got = run_attn(ln, q, c, table, q_len, kv_len, window, cells=cells).cpu().numpy()
    check_attn(got, q, q_len, kv_len, keys, vals, window)
    assert np.array_equal(got, run_attn(ln, q, c, table, q_len, kv_len, window, cells=cells).cpu().numpy())


@pytest.mark.parametrize("qscale,kstd,vstd", [(1e-6, 1.0, 1.0), (30.0, 1.0, 1.0), (1.0, 1e-3, 1e-3),
                                              (1e4, 1e-4, 500.0), (1.0, 20.0, 8000.0), (1e-30, 1.0, 1e-2)])
@pytest.mark.parametrize("q_len,kv_len,cells", [([1], [200], 0), ([100], [180], 0), ([100], [180], 1 << 14), ([130], [180], 1 << 14)])
def test_attention_of_small_and_large_values(ln, qscale, kstd, vstd, q_len, kv_len, cells):
    rng = np.random.default_rng(11)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, 32, 8, 2, 64, qscale, kstd, vstd)
    got = run_attn(ln, q, c, table, q_len, kv_len, cells=cells).cpu().numpy()
    check_attn(got, q, q_len, kv_len, keys, vals)


@pytest.mark.parametrize("q_len,cells", [([1], 0), ([90], 0), ([90], 1 << 14), ([260], 1 << 14)])
def test_attention_is_exact_where_one_cell_counts(ln, q_len, cells):
    """Zero queries weigh all cells alike; equal values come out as they are, to 22 bits; and every
    code of the half range, as the value of the only cell, comes out as its real number."""
    page, nkv, hd = 16, 2, 64
    codes = np.arange(0x4000 - 24 * 128, 0x4800, dtype=np.uint16)
    codes = np.concatenate([codes, codes | 0x8000, [0, 0x8000]]).astype(np.uint16)
    for i in range(0, len(codes), nkv * hd):
        v = np.resize(codes[i:i + nkv * hd], (1, nkv, hd))
        n = q_len[0]
        c = R.Cache(20, page, nkv, hd, fill=0)
        row = np.arange(18)
        c.put(row, np.arange(n), np.zeros((n, nkv, hd), np.uint16), np.repeat(v, n, 0))
        q = np.zeros((n, 4, hd), np.float32)
        got = run_attn(ln, q, c, row[None].astype(np.int32), q_len, q_len, cells=cells).cpu().numpy()
        want = np.repeat(R.value(v), 2, 1)
        # values: 2^-22 as halves, 2^-23 of the power; below the normal halves 2^-36; the mean of n
        # equal terms: n 2^-23
        tol = np.abs(want) * (2.0 ** -21 + n * 2.0 ** -23) + 2.0 ** -35
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("q_len,kv_len,cells", [([4, 3], [2, 3], 0), ([40, 1], [10, 0], 0), ([5, 90], [-3, 30], 0),
                                                ([5, 90], [-3, 30], 1 << 14), ([5, 380], [-3, 300], 1 << 13)])
def test_rows_without_cells_are_zero(ln, q_len, kv_len, cells):
    rng = np.random.default_rng(12)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, 16, 6, 2, 64)
    got = run_attn(ln, q, c, table, q_len, kv_len, cells=cells).cpu().numpy()
    pos = np.concatenate(positions(q_len, kv_len))
    assert (got[pos < 0] == 0).all() and np.isfinite(got).all()
    check_attn(got, q, q_len, kv_len, keys, vals)


@pytest.mark.parametrize("q_len,kv_len,cells", [([1], [900], 0), ([77], [300], 0), ([77], [300], 1 << 14), ([140], [300], 1 << 14)])
def test_bad_pages_hide_their_cells(ln, q_len, kv_len, cells):
    rng = np.random.default_rng(13)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, 16, 8, 2, 64)
    index_error(ln)
    table[0, 3], table[0, 5] = -7, c.n_pages
    got = run_attn(ln, q, c, table, q_len, kv_len, cells=cells).cpu().numpy()
    assert index_error(ln)[0] == 1 and index_error(ln)[0] == 0
    check_attn(got, q, q_len, kv_len, keys, vals, hidden=set(range(48, 64)) | set(range(80, 96)))


def test_cells_past_the_table_are_hidden(ln):
    rng = np.random.default_rng(14)
    q, c, table, keys, vals = attn_case(rng, [2], [64], 16, 2, 1, 32)
    index_error(ln)
    got = run_attn(ln, q, c, table[:, :3], [2], [64]).cpu().numpy()
    assert index_error(ln)[0] == 1
    check_attn(got, q, [2], [64], [keys[0]], [vals[0]], hidden=set(range(48, 64)))


@pytest.mark.parametrize("q_len,kv_len,cells", [([1, 2], [700, 40], 0), ([80, 90], [300, 90], 0), ([80, 90], [300, 90], 1 << 14),
                                                ([280, 90], [300, 90], 1 << 14)])
def test_rows_of_no_sequence_strides_and_in_place(ln, q_len, kv_len, cells):
    rng = np.random.default_rng(15)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, 16, 6, 2, 64, width=60)
    T, first, table = sum(q_len), 3, widen(table, 16, cells)
    buf = torch.full((T + 8, 6 * 64 + 5), 9.0, device="cuda")
    view = torch.as_strided(buf, (T + 8, 6, 64), (6 * 64 + 5, 64, 1), 2)
    view[first:first + T] = dev(q)
    args = (dev(c.k), dev(c.v), c.page, dev(table), dev(starts(q_len, first)), dev(np.int32(kv_len)), 0.125)
    out = torch.full((T + 8, 6, 64), 9.0, device="cuda")
    ln.paged.attention(view, *args, out=out)
    o = out.cpu().numpy()
    check_attn(o[first:first + T], q, q_len, kv_len, keys, vals)
    assert (o[:first] == 9).all() and (o[first + T:] == 9).all()
    ln.paged.attention(view, *args, out=view)                         # dst is q
    assert torch.equal(view, out)
    rest = buf.clone()
    torch.as_strided(rest, (T + 8, 6, 64), (6 * 64 + 5, 64, 1), 2)[:] = 9.0
    assert (rest == 9).all()


@pytest.mark.parametrize("q_len,kv_len,cells", [([1], [500], 0), ([70], [140], 0), ([70], [140], 1 << 15), ([270], [340], 1 << 14)])
def test_infinities_and_nan(ln, q_len, kv_len, cells):
    """A NaN or infinite query gives its own row alone no numbers."""
    rng = np.random.default_rng(16)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, 16, 4, 2, 64)
    want = run_attn(ln, q, c, table, q_len, kv_len, cells=cells).cpu().numpy()
    q2 = q.copy()
    q2[0, 1, 5] = np.nan
    q2[0, 2, 7] = np.inf
    got = run_attn(ln, q2, c, table, q_len, kv_len, cells=cells).cpu().numpy()
    assert np.isnan(got[0, 1]).all() and np.isnan(got[0, 2]).all()
    keep = np.ones(got.shape[:2], bool)
    keep[0, 1] = keep[0, 2] = False
    assert np.array_equal(got[keep], want[keep])


def test_pages_past_32_bits(ln):
    """Page offsets beyond 2^31 codes, keys and values."""
    page, nkv, hd = 256, 8, 256
    n_pages = (1 << 31) // (page * nkv * hd) + 24
    k, v = ln.paged.alloc_pages(n_pages, page, nkv, hd)
    rng = np.random.default_rng(17)
    n = 2 * page
    ids = np.int32([[n_pages - 1, n_pages - 3]])
    x = rng.standard_normal((n, nkv, 2, hd)).astype(np.float32)
    xd = dev(x)
    q = (rng.standard_normal((n, 8, hd))).astype(np.float32)
    st, kl, tb = dev(np.int32([0, n])), dev(np.int32([n])), dev(ids)
    ln.paged.rope_store_kv(None, xd[:, :, 0].contiguous(), xd[:, :, 1].contiguous(), k, v, page, tb, st, kl, None,
                           n_dims=0)
    rows = [0, 200, n - 1]
    got = ln.paged.attention(dev(q), k, v, page, tb, st, kl, hd ** -0.5).cpu().numpy()[rows]
    kc, vc = R.store_codes(x[:, :, 0]), R.store_codes(x[:, :, 1])
    ref, tol = R.attention(q[rows], kc, vc, np.array(rows), hd ** -0.5)
    assert (np.abs(got - ref) <= tol).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 7, 31, 97, 250, 255, 256])
def test_a_pool_of_one_page(ln, hd, n):
    """The only page is the last one of the pool: loads ahead of the last cells stay inside it."""
    rng = np.random.default_rng(n)
    for q_len in (1, min(n, 70)):
        c = R.Cache(1, 256, 2, hd)
        keys, vals = (R.store_codes(rng.standard_normal((n, 2, hd)).astype(np.float32)) for _ in range(2))
        c.put([0], np.arange(n), keys, vals)
        q = rng.standard_normal((q_len, 4, hd)).astype(np.float32)
        got = run_attn(ln, q, c, np.int32([[0]]), [q_len], [n]).cpu().numpy()
        check_attn(got, q, [q_len], [n], [keys], [vals])


def test_long_cache_of_one_token(ln):
    """Many splits: the parts of a long cache are joined."""
    rng = np.random.default_rng(18)
    for n in (4096, 20011):
        q, c, table, keys, vals = attn_case(rng, [1], [n], 64, 4, 2, 64)
        got = run_attn(ln, q, c, table, [1], [n]).cpu().numpy()
        check_attn(got, q, [1], [n], keys, vals)
        # the same cells under a table of far more pages: other splits
        wide = np.full((1, 4 * table.shape[1]), -1, np.int32)
        wide[:, :table.shape[1]] = table
        got = run_attn(ln, q, c, wide, [1], [n]).cpu().numpy()
        check_attn(got, q, [1], [n], keys, vals)


@pytest.mark.parametrize("window", [1, 63, 64, 65, 500, 513, 1000, 5000, 1 << 40])
def test_windows_of_single_tokens(ln, window):
    """Parts are as many as a window may need: windows of any length behind long caches."""
    rng = np.random.default_rng(23)
    kv_len = [4096, 3000, 1, 77]
    q, c, table, keys, vals = attn_case(rng, [1] * 4, kv_len, 16, 8, 2, 64)
    got = run_attn(ln, q, c, table, [1] * 4, kv_len, window).cpu().numpy()
    check_attn(got, q, [1] * 4, kv_len, keys, vals, window)


# ---- together ----------------------------------------------------------------------------

def test_chunks_and_single_tokens_agree(ln):
    """A prompt stored and attended in chunks, or token by token: the same cells, bit for bit, and the
    same attention within the bound of both."""
    rng = np.random.default_rng(19)
    nh, nkv, hd, page, n = 6, 2, 64, 16, 75
    x = rng.standard_normal((n, nh + 2 * nkv, hd)).astype(np.float32)
    xd, cs = dev(x), dev(rope_table(ln, 128, hd))
    table, n_pages = R.tables(rng, [n], page)
    caches = []
    for chunks in ([n], [1] * n, [40, 1, 33, 1]):
        k, v = ln.paged.alloc_pages(n_pages, page, nkv, hd)
        outs, at = [], 0
        for m in chunks:
            st, kl = dev(np.int32([0, m])), dev(np.int32([at + m]))
            part = xd[at:at + m]
            q = ln.paged.rope_store_kv(part[:, :nh], part[:, nh:nh + nkv], part[:, nh + nkv:], k, v, page, dev(table), st,
                                       kl, cs)
            outs.append(ln.paged.attention(q, k, v, page, dev(table), st, kl, hd ** -0.5))
            at += m
        caches.append((k, v, torch.cat(outs).cpu().numpy()))
    c = R.Cache(n_pages, page, nkv, hd)
    c.k, c.v = (t.cpu().numpy().view(np.uint16) for t in caches[0][:2])
    keys, vals = c.get(table[0], n)
    rot = R.rope(x[:, :nh], rope_table(ln, 128, hd)[:n], False, hd)
    ref, tol = R.attention(rot, keys, vals, np.arange(n), hd ** -0.5)
    for k, v, o in caches:
        assert torch.equal(k, caches[0][0]) and torch.equal(v, caches[0][1])
        assert (np.abs(o - ref) <= tol).all()


def test_captured_steps_replay_with_their_lengths(ln):
    """A step (store, attention, draw) captured once; replays with other lengths, pages and inputs,
    with eager work and synchronizations between, equal the eager step every time."""
    rng = np.random.default_rng(20)
    nh, nkv, hd, page, S, W = 6, 2, 64, 16, 5, 40
    cs = dev(rope_table(ln, W * page, hd))
    k, v = ln.paged.alloc_pages(S * W, page, nkv, hd)
    k.random_(0x3c00, 0x4200)
    v.random_(0x3c00, 0x4200)
    qkv = torch.zeros((S, nh + 2 * nkv, hd), device="cuda")
    table = torch.zeros((S, W), dtype=torch.int32, device="cuda")
    start, kvl = dev(np.arange(S + 1, dtype=np.int32)), torch.ones(S, dtype=torch.int32, device="cuda")
    u = torch.zeros(S, device="cuda")

    def step():
        q = ln.paged.rope_store_kv(qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:], k, v, page, table, start, kvl, cs)
        o = ln.paged.attention(q, k, v, page, table, start, kvl, 0.125)
        return q, o, *ln.sample(o.view(S, -1) * 20, u)

    def inputs():
        qkv.copy_(dev(rng.standard_normal(qkv.shape).astype(np.float32)))
        table.copy_(dev(rng.permutation(S * W).astype(np.int32).reshape(S, W)))
        kvl.copy_(dev(rng.integers(1, W * page, S).astype(np.int32)))
        u.copy_(dev(rng.random(S).astype(np.float32)))

    inputs()
    step()
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            got = step()
    torch.cuda.current_stream().wait_stream(s)
    for i in range(5):
        inputs()
        g.replay()
        have = [t.clone() for t in got]
        if i % 2:
            torch.cuda.synchronize()
        want = step()
        for a, b in zip(have, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("hd,q_len,cells", [(64, 100, 16384), (64, 150, 8192), (128, 100, 8192), (128, 600, 4096)])
def test_captured_chunks_replay_with_their_lengths(ln, hd, q_len, cells):
    """Chunks' kernels (decoding in each workgroup, and before them all) in a captured graph."""
    rng = np.random.default_rng(22)
    k, v = ln.paged.alloc_pages(cells // 16, 16, 2, hd)
    k.random_(0x3c00, 0x4200)
    v.random_(0x3c00, 0x4200)
    q = torch.randn((q_len, 8, hd), device="cuda")
    table = torch.zeros((1, cells // 16), dtype=torch.int32, device="cuda")
    start, kvl = dev(np.int32([0, q_len])), dev(np.int32([q_len]))

    def inputs(n):
        table.copy_(dev(rng.permutation(cells // 16).astype(np.int32)[None]))
        kvl.fill_(n)
        q.copy_(torch.randn((q_len, 8, hd), device="cuda"))

    inputs(q_len)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            got = ln.paged.attention(q, k, v, 16, table, start, kvl, 0.1)
    for n in (q_len + 50, 3000, q_len, q_len - 30):
        inputs(n)
        g.replay()
        have = got.clone()
        if n % 100:
            torch.cuda.synchronize()
        assert torch.equal(have, ln.paged.attention(q, k, v, 16, table, start, kvl, 0.1)), n


def test_two_streams_at_once(ln):
    """Calls on two streams, each with its own workspace, beside each other."""
    rng = np.random.default_rng(21)
    cases = [attn_case(rng, [1, 1], [3000, 2000], 16, 8, 2, 64), attn_case(rng, [2, 1], [1500, 2900], 32, 8, 2, 64)]
    lens = [([1, 1], [3000, 2000]), ([2, 1], [1500, 2900])]
    d = [(dev(q), dev(c.k), dev(c.v), c.page, dev(t), dev(starts(n[0])), dev(np.int32(n[1])), 0.125)
         for (q, c, t, _, _), n in zip(cases, lens)]
    want = [ln.paged.attention(*a) for a in d]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in d]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ln.paged.attention(*d[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
