"""The paged xlns16 cache on the GPU: calls that a serving loop makes beside those of
test_gpu_paged.py, against the same 64-bit form and bounds."""
import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import attn_case, check_attn, dev, index_error, positions, rope_table, run_attn, starts

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ln():
    import lnship
    import lnship.paged
    lnship.init()
    return lnship


# ---- rotation in place -------------------------------------------------------------------

@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("T,nh,nkv,hd,nd", [
    (1, 1, 1, 8, 8), (3, 9, 3, 64, 64), (5, 4, 2, 80, 80), (7, 6, 2, 96, 96), (20, 32, 8, 128, 128), (9, 3, 3, 256, 256),
    (6, 5, 1, 72, 18), (11, 3, 1, 136, 64), (4, 2, 2, 24, 0), (300, 3, 1, 256, 250),
    # 2^19 values and more: the other kernel
    (700, 4, 2, 128, 128), (1500, 4, 2, 80, 64)])
def test_queries_rotated_in_place(ln, T, nh, nkv, hd, nd, neox):
    """out = q, of its own or within the rows of a fused product: queries and cells bit for bit, and
    nothing else written."""
    print(f"\n[store] in place {T} x {nh}/{nkv}x{hd} rot {nd} neox {neox}", flush=True)
    rng = np.random.default_rng(hd + T)
    page = 32
    x = rng.standard_normal((T, nh + 2 * nkv, hd)).astype(np.float32)
    cs = rope_table(ln, T + 3, nd) if nd else None
    table, n_pages = R.tables(rng, [T + 3], page)
    batch = (page, dev(table), dev(starts([T])), dev(np.int32([T + 3])), dev(cs) if nd else None)
    rot = R.rope(x[:, :nh + nkv], cs[3:], neox, nd) if nd else x[:, :nh + nkv]
    c = R.Cache(n_pages, page, nkv, hd, fill=0)
    c.put(table[0], np.arange(3, T + 3), R.store_codes(rot[:, nh:]), R.store_codes(x[:, nh + nkv:]))
    for fused in (True, False):
        xd = dev(x)
        q = xd[:, :nh] if fused else xd[:, :nh].contiguous()
        k, v = ln.paged.alloc_pages(n_pages, page, nkv, hd)
        got = ln.paged.rope_store_kv(q, xd[:, nh:nh + nkv], xd[:, nh + nkv:], k, v, *batch, n_dims=nd, neox=neox, out=q)
        assert got is q and np.array_equal(q.cpu().numpy().view(np.uint32), rot[:, :nh].view(np.uint32))
        assert np.array_equal(xd[:, nh:].cpu().numpy(), x[:, nh:])
        assert np.array_equal(k.cpu().numpy().view(np.uint16), c.k) and np.array_equal(v.cpu().numpy().view(np.uint16), c.v)

def test_outputs_that_overlap_inputs_are_refused(ln):
    """Shifted or otherwise strided views of q, and k or v, as out; nothing is written."""
    T, nh, nkv, hd = 3, 2, 1, 32
    k, v = ln.paged.alloc_pages(2, 16, nkv, hd)
    batch = (16, dev(np.int32([[0, 1]])), dev(np.int32([0, T])), dev(np.int32([T])))
    buf = torch.ones(T * 5 * hd + 64, device="cuda")
    q = torch.as_strided(buf, (T, nh, hd), (4 * hd, hd, 1), 0)
    x = torch.ones((T, 2 * nkv, hd), device="cuda")
    for out in (torch.as_strided(buf, (T, nh, hd), (4 * hd, hd, 1), hd), torch.as_strided(buf, (T, nh, hd), (5 * hd, hd, 1), 0)):
        with pytest.raises(ln.LnshipError, match="overlaps q"):
            ln.paged.rope_store_kv(q, x[:, :1], x[:, 1:], k, v, *batch, None, n_dims=0, out=out)
        with pytest.raises(ln.LnshipError, match="overlaps q"):
            ln.paged.attention(q, k, v, *batch, 1.0, out=out)
    wide = torch.ones((T, nh + 2 * nkv, hd), device="cuda")
    for at in (1, 2):
        with pytest.raises(ln.LnshipError, match="overlaps k or v"):
            ln.paged.rope_store_kv(q, wide[:, 2:3], wide[:, 3:], k, v, *batch, None, n_dims=0, out=wide[:, at:at + nh])
    torch.cuda.synchronize()
    assert (buf == 1).all() and (wide == 1).all() and not k.any() and not v.any()
    # in the gaps of q's rows, and of the fused rows
    gap = torch.as_strided(buf, (T, nh, hd), (4 * hd, hd, 1), 2 * hd)
    ln.paged.attention(q, k, v, *batch, 1.0, out=gap)
    assert (gap == 0).all() and (q == 1).all()


# ---- pages behind a window ---------------------------------------------------------------

FREED = [
    # q_len, kv_len, page, heads, kv heads, dim, window, cells of the table
    ([1], [1000], 16, 12, 4, 64, 33, 0),
    ([1, 1, 1], [1000, 517, 40], 32, 8, 2, 128, 100, 0),
    ([1] * 40, [300 + 29 * i for i in range(40)], 16, 16, 8, 128, 65, 0),
    ([9, 3], [700, 400], 16, 4, 2, 200, 50, 0),
    ([40, 90], [300, 400], 16, 4, 2, 64, 17, 1 << 14),
    ([70], [700], 32, 8, 2, 128, 111, 1 << 14),
    ([520], [900], 16, 8, 2, 64, 200, 1 << 13),
    ([600, 300], [1200, 1111], 32, 4, 2, 128, 77, 1 << 13),
]


@pytest.mark.parametrize("q_len,kv_len,page,nh,nkv,hd,window,cells", FREED)
def test_pages_behind_the_window_may_be_freed(ln, q_len, kv_len, page, nh, nkv, hd, window, cells):
    """A page whose cells no new token sees is not looked at: its number may be -1, and is no error."""
    print(f"\n[attn] {q_len} {kv_len} page {page} {nh}/{nkv}x{hd} window {window} freed", flush=True)
    rng = np.random.default_rng(window)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, page, nh, nkv, hd)
    want = run_attn(ln, q, c, table, q_len, kv_len, window, cells=cells).cpu().numpy()
    first = [max(0, m - n - window + 1) // page for n, m in zip(q_len, kv_len)]
    assert any(first)
    for s, f in enumerate(first):
        table[s, :f] = -1
    index_error(ln)
    got = run_attn(ln, q, c, table, q_len, kv_len, window, cells=cells).cpu().numpy()
    assert index_error(ln)[0] == 0
    assert np.array_equal(got, want)
    check_attn(got, q, q_len, kv_len, keys, vals, window)
    # the first page that is seen counts
    s = int(np.argmax(first))
    table[s, first[s]] = -5
    run_attn(ln, q, c, table, q_len, kv_len, window, cells=cells)
    assert index_error(ln) == (1, -5)


# ---- many sequences ----------------------------------------------------------------------

def many(rng, n_seq, most, past):
    """Lengths of n_seq sequences, some without new tokens, those beside multiples of 64 and 79 among them."""
    q_len = rng.integers(0, most + 1, n_seq)
    for at in (0, 63, 64, 65, 79, 128, 4095, 4096, n_seq - 1):
        q_len[min(at, n_seq - 1)] = at % 2
    q_len[n_seq // 2] = most
    return q_len.tolist(), (q_len + rng.integers(0, past, n_seq)).tolist()


def check_some(got, q, q_len, kv_len, keys, vals, rng, window=0):
    """check_attn of sequences drawn at random and of those at the ends of a search's rounds."""
    n_seq, at = len(q_len), np.concatenate([[0], np.cumsum(q_len)])
    some = set(rng.choice(n_seq, min(n_seq, 60), replace=False).tolist())
    some |= {s for b in (0, 64, 79, 128, 4096, n_seq) for s in (b - 1, b, b + 1) if 0 <= s < n_seq}
    for s in some:
        check_attn(got[at[s]:at[s + 1]], q[at[s]:at[s + 1]], [q_len[s]], [kv_len[s]], [keys[s]], [vals[s]], window)


@pytest.mark.parametrize("n_seq,most,nh,nkv,hd,cells", [
    (64, 3, 4, 2, 64, 0), (65, 3, 4, 2, 64, 0), (129, 3, 4, 2, 128, 0), (300, 1, 32, 8, 64, 0), (5000, 2, 2, 1, 8, 0),
    # chunks: each workgroup decodes; decoded before
    (65, 20, 8, 1, 16, 1 << 13), (130, 10, 32, 2, 72, 1 << 11), (4200, 2, 128, 1, 8, 1 << 9),
    (70, 20, 64, 1, 8, 1 << 10), (129, 16, 64, 1, 40, 1 << 10)])
def test_attention_of_many_sequences(ln, n_seq, most, nh, nkv, hd, cells):
    print(f"\n[attn] {n_seq} sequences of up to {most} tokens, {nh}/{nkv}x{hd}, {cells} cells", flush=True)
    rng = np.random.default_rng(n_seq + hd)
    q_len, kv_len = many(rng, n_seq, most, 60)
    q, c, table, keys, vals = attn_case(rng, q_len, kv_len, 16, nh, nkv, hd)
    for window in (0, 21):
        got = run_attn(ln, q, c, table, q_len, kv_len, window, cells=cells).cpu().numpy()
        assert np.isfinite(got).all()
        check_some(got, q, q_len, kv_len, keys, vals, rng, window)


@pytest.mark.parametrize("n_seq,hd", [(64, 8), (65, 8), (129, 64), (1000, 16), (5000, 8)])
def test_stores_of_many_sequences(ln, n_seq, hd):
    """Fewer than 2^19 values: the kernel that looks a row's sequence up with a wave."""
    print(f"\n[store] {n_seq} sequences x {hd}", flush=True)
    rng = np.random.default_rng(n_seq)
    q_len, kv_len = many(rng, n_seq, 3, 40)
    T, page = sum(q_len), 16
    assert T * 3 * hd < 1 << 19
    x = rng.standard_normal((T, 3, hd)).astype(np.float32)
    cs = rope_table(ln, max(kv_len) + 1, hd)
    table, n_pages = R.tables(rng, kv_len, page)
    k, v = ln.paged.alloc_pages(n_pages, page, 1, hd)
    xd = dev(x)
    out = ln.paged.rope_store_kv(xd[:, :1], xd[:, 1:2], xd[:, 2:], k, v, page, dev(table), dev(starts(q_len)),
                                 dev(np.int32(kv_len)), dev(cs))
    pos = positions(q_len, kv_len)
    rot = R.rope(x[:, :2], cs[np.concatenate(pos)], False, hd)
    kc, vc = R.store_codes(rot[:, 1:]), R.store_codes(x[:, 2:])
    c = R.Cache(n_pages, page, 1, hd, fill=0)
    at = 0
    for s, p in enumerate(pos):
        c.put(table[s], p, kc[at:at + len(p)], vc[at:at + len(p)])
        at += len(p)
    assert np.array_equal(out.cpu().numpy().view(np.uint32), rot[:, :1].view(np.uint32))
    assert np.array_equal(k.cpu().numpy().view(np.uint16), c.k) and np.array_equal(v.cpu().numpy().view(np.uint16), c.v)
