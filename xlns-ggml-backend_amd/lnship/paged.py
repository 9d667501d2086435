"""The paged xlns16 KV cache of several sequences: pages, their use by a batch
of new tokens, and the two operators over them (include/lnship.h:
lnship16_rope_store_kv_paged, lnship16_attn_paged).

A batch is described by device tensors (int32), so that a captured graph
replays with other lengths and pages: q_start [n_seq + 1] (rows q_start[s] to
q_start[s+1] - 1 are sequence s's new tokens), kv_len [n_seq] (its cells, the
new tokens' included) and table [n_seq, pages a sequence may have].
"""
import struct

import torch

from . import LnshipError, check, current_stream, lib

# The fields of PagedKV, PagedStoreArgs and PagedAttnArgs, packed: a tenth of
# the time that the structures take, of calls that every layer of a step makes.
_KV, _STORE, _ATTN = (struct.Struct(f) for f in ("PPqqqqPqqqPP", "PPPqqqqiiPqPq", "PPqqqfqPN"))

_I16, _I32, _F32 = torch.int16, torch.int32, torch.float32


def alloc_pages(n_pages, page, n_head_kv, head_dim, device="cuda"):
    """Key and value pages of one layer, empty: int16 [n_pages, n_head_kv, page * head_dim] each."""
    shape = (n_pages, n_head_kv, page * head_dim)
    return tuple(torch.zeros(shape, dtype=torch.int16, device=device) for _ in range(2))


def _no(what):
    raise LnshipError("paged cache: " + what)


def _kv(k_pages, v_pages, page, table, q_start, kv_len, ntok):
    """lnship_paged_kv of the tensors, checked, as bytes; the device that all must be on, the current one;
    n_head_kv and head_dim."""
    dev = k_pages.get_device()
    shape = k_pages.shape
    if k_pages.dtype is not _I16 or k_pages.dim() != 3 or not k_pages.is_contiguous():
        _no("k_pages must be contiguous int16 [n_pages, n_head_kv, page * head_dim]")
    if v_pages.dtype is not _I16 or v_pages.shape != shape or not v_pages.is_contiguous() or v_pages.get_device() != dev:
        _no("v_pages must be as k_pages")
    n_seq = kv_len.numel()
    if kv_len.dtype is not _I32 or kv_len.dim() != 1 or not kv_len.is_contiguous() or kv_len.get_device() != dev:
        _no("kv_len must be contiguous int32 [n_seq] on the pages' device")
    if q_start.dtype is not _I32 or q_start.shape != (n_seq + 1,) or not q_start.is_contiguous() or \
            q_start.get_device() != dev:
        _no("q_start must be contiguous int32 [n_seq + 1] on the pages' device")
    if table.dtype is not _I32 or table.dim() != 2 or not table.is_contiguous() or table.get_device() != dev:
        _no("table must be contiguous int32 [n_seq, pages] on the pages' device")
    rows, width = table.shape
    n_pages, n_head_kv, codes = shape
    if rows != n_seq:
        _no("table must have a row for every sequence")
    if page < 1 or codes % page:
        _no("pages of %d codes a head hold no %d cells" % (codes, page))
    hd = codes // page
    return _KV.pack(k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page, n_head_kv, hd, table.data_ptr(), width, ntok,
                    n_seq, q_start.data_ptr(), kv_len.data_ptr()), dev, n_head_kv, hd


def _ld(t, name, ntok, heads, dim, dev):
    """The row stride of a [ntok, heads, dim] float32 tensor whose heads lie behind each other."""
    if t.dtype is not _F32 or t.shape != (ntok, heads, dim) or t.get_device() != dev:
        _no("%s must be float32 [%d, %d, %d] on the pages' device" % (name, ntok, heads, dim))
    s0, s1, s2 = t.stride()
    if s2 != 1 or (s1 != dim and heads > 1):
        _no(name + ": a row's heads must lie behind each other")
    if ntok > 1 and s0 < heads * dim:
        _no(name + ": rows must not overlap")
    return s0 if ntok > 1 else max(s0, heads * dim)


def _apart(a, a_ld, a_w, b, b_ld, b_w, n):
    """Whether n rows of a_w floats from address a on, a_ld floats apart, share no memory with n of b's: of
    rows equally far apart, one may lie in the gaps of the other."""
    if a + ((n - 1) * a_ld + a_w) * 4 <= b or b + ((n - 1) * b_ld + b_w) * 4 <= a:
        return True
    d = (b - a) % (a_ld * 4)
    return a_ld == b_ld and a_w * 4 <= d <= (a_ld - b_w) * 4


def rope_store_kv(q, k, v, k_pages, v_pages, page, table, q_start, kv_len, cos_sin, n_dims=None, neox=False, out=None):
    """Rotates the new tokens' queries and keys and stores their keys and
    values into the pages (in place).  q [ntok, n_head, head_dim] (or None), k,
    v [ntok, n_head_kv, head_dim] float32: arrays, or the parts of a fused
    q|k|v product's rows; cos_sin [n_pos, n_dims / 2, 2] float32 (None with
    n_dims 0: nothing is rotated).  Returns the rotated queries.  out may be q."""
    ntok = k.shape[0]
    kv, dev, nkv, hd = _kv(k_pages, v_pages, page, table, q_start, kv_len, ntok)
    stream = current_stream(dev)
    if n_dims is None:
        n_dims = hd if cos_sin is not None else 0
    cs = n_pos = 0
    if n_dims:
        if cos_sin is None or cos_sin.dtype is not _F32 or cos_sin.dim() != 3 or not cos_sin.is_contiguous() or \
                cos_sin.get_device() != dev or cos_sin.shape[1:] != (n_dims // 2, 2):
            _no("cos_sin must be contiguous float32 [n_pos, n_dims / 2, 2] on the pages' device")
        cs, n_pos = cos_sin.data_ptr(), cos_sin.shape[0]
    nh = q_ld = out_ld = q_at = out_at = 0
    k_at, v_at, k_ld, v_ld = k.data_ptr(), v.data_ptr(), _ld(k, "k", ntok, nkv, hd, dev), _ld(v, "v", ntok, nkv, hd, dev)
    if q is not None:
        nh = q.shape[1]
        given = out is not None
        if not given:
            out = torch.empty((ntok, nh, hd), dtype=_F32, device=k_pages.device)
        q_ld, out_ld = _ld(q, "q", ntok, nh, hd, dev), _ld(out, "out", ntok, nh, hd, dev)
        q_at, out_at = q.data_ptr(), out.data_ptr()
        if given and ntok and not (_apart(out_at, out_ld, nh * hd, k_at, k_ld, nkv * hd, ntok) and
                                   _apart(out_at, out_ld, nh * hd, v_at, v_ld, nkv * hd, ntok)):
            _no("out overlaps k or v")
    a = _STORE.pack(q_at, k_at, v_at, q_ld, k_ld, v_ld, nh, n_dims, neox, cs, n_pos, out_at, out_ld)
    check(lib().lnship16_rope_store_kv_paged(kv, a, stream))
    return out


def attention(q, k_pages, v_pages, page, table, q_start, kv_len, scale, window=0, out=None):
    """Attention of the new tokens q [ntok, n_head, head_dim] float32 over
    their sequences' cells in the pages: those up to each token's own position
    and, with window > 0, no further than window - 1 before it (pages behind
    every new token's window are not looked at, and may be freed).  Returns
    out, [ntok, n_head, head_dim] float32, which may be q.  Its workspace, up
    to 1 GiB for prompts, comes from torch's allocator."""
    ntok, nh = q.shape[:2]
    kv, dev, _, hd = _kv(k_pages, v_pages, page, table, q_start, kv_len, ntok)
    stream = current_stream(dev)
    if out is None:
        out = torch.empty((ntok, nh, hd), dtype=_F32, device=k_pages.device)
    q_ld, out_ld = _ld(q, "q", ntok, nh, hd, dev), _ld(out, "out", ntok, nh, hd, dev)
    L = lib()
    need = L.lnship16_attn_paged_work(kv, nh)
    if need < 0:
        check(need)
    # (of torch's allocator: the stream's own, a captured graph's own)
    work = torch.empty(need, dtype=torch.uint8, device=k_pages.device) if need else None
    a = _ATTN.pack(q.data_ptr(), out.data_ptr(), q_ld, out_ld, nh, scale, window, work.data_ptr() if need else 0, need)
    check(L.lnship16_attn_paged(kv, a, stream))
    return out
