"""The paged xlns16 KV cache of several sequences: pages, their use by a batch
of new tokens, and the two operators over them (include/lnship.h:
lnship16_rope_store_kv_paged, lnship16_attn_paged).

A batch is described by device tensors (int32), so that a captured graph
replays with other lengths and pages: q_start [n_seq + 1] (rows q_start[s] to
q_start[s+1] - 1 are sequence s's new tokens), kv_len [n_seq] (its cells, the
new tokens' included) and table [n_seq, pages a sequence may have].
"""
import ctypes

from . import LnshipError, PagedAttnArgs, PagedKV, PagedStoreArgs, _stream, check, init, lib


def alloc_pages(n_pages, page, n_head_kv, head_dim, device="cuda"):
    """Key and value pages of one layer, empty: int16 [n_pages, n_head_kv, page * head_dim] each."""
    import torch
    shape = (n_pages, n_head_kv, page * head_dim)
    return tuple(torch.zeros(shape, dtype=torch.int16, device=device) for _ in range(2))


def _need(ok, what):
    if not ok:
        raise LnshipError("paged cache: " + what)


def _kv(k_pages, v_pages, page, table, q_start, kv_len, ntok):
    import torch
    dev = k_pages.device
    _need(k_pages.is_cuda and dev.index == torch.cuda.current_device(), "the pages are not on the current device")
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        _need(t.dtype == torch.int16 and t.dim() == 3 and t.is_contiguous() and t.shape == k_pages.shape and
              t.device == dev, name + " must be contiguous int16 [n_pages, n_head_kv, page * head_dim]")
    for t, name in ((table, "table"), (q_start, "q_start"), (kv_len, "kv_len")):
        _need(t.dtype == torch.int32 and t.device == dev, name + " must be int32 on the pages' device")
    n_seq = kv_len.shape[0]
    _need(kv_len.dim() == 1 and kv_len.is_contiguous(), "kv_len must be contiguous [n_seq]")
    _need(q_start.shape == (n_seq + 1,) and q_start.is_contiguous(), "q_start must be contiguous [n_seq + 1]")
    _need(table.dim() == 2 and table.shape[0] == n_seq and table.is_contiguous(),
          "table must be contiguous [n_seq, pages]")
    n_pages, n_head_kv, codes = k_pages.shape
    _need(page > 0 and codes % page == 0, "pages of %d codes a head hold no %d cells" % (codes, page))
    return PagedKV(k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page, n_head_kv, codes // page, table.data_ptr(),
                   table.shape[1], ntok, n_seq, q_start.data_ptr(), kv_len.data_ptr())


def _rows(t, name, ntok, heads, dim, dev):
    """The row stride of a [ntok, heads, dim] float32 tensor whose heads lie behind each other."""
    import torch
    _need(t.dtype == torch.float32 and t.shape == (ntok, heads, dim) and t.device == dev,
          "%s must be float32 [%d, %d, %d] on the pages' device" % (name, ntok, heads, dim))
    s = t.stride()
    _need(s[2] == 1 and (s[1] == dim or heads == 1), name + ": a row's heads must lie behind each other")
    return s[0] if ntok > 1 else max(s[0], heads * dim)


def rope_store_kv(q, k, v, k_pages, v_pages, page, table, q_start, kv_len, cos_sin, n_dims=None, neox=False, out=None):
    """Rotates the new tokens' queries and keys and stores their keys and
    values into the pages (in place).  q [ntok, n_head, head_dim] (or None), k,
    v [ntok, n_head_kv, head_dim] float32: arrays, or the parts of a fused
    q|k|v product's rows; cos_sin [n_pos, n_dims / 2, 2] float32 (None with
    n_dims 0: nothing is rotated).  Returns the rotated queries."""
    import torch
    init()
    ntok = k.shape[0]
    kv = _kv(k_pages, v_pages, page, table, q_start, kv_len, ntok)
    dev, hd, nkv = k_pages.device, kv.head_dim, kv.n_head_kv
    if n_dims is None:
        n_dims = hd if cos_sin is not None else 0
    _need(n_dims == 0 or (cos_sin is not None and cos_sin.dtype == torch.float32 and cos_sin.dim() == 3 and
                          cos_sin.shape[1:] == (n_dims // 2, 2) and cos_sin.is_contiguous() and
                          cos_sin.device == dev), "cos_sin must be contiguous float32 [n_pos, n_dims / 2, 2]")
    nh = q.shape[1] if q is not None else 0
    if nh and out is None:
        out = torch.empty((ntok, nh, hd), dtype=torch.float32, device=dev)
    a = PagedStoreArgs(q.data_ptr() if nh else None, k.data_ptr(), v.data_ptr(),
                       _rows(q, "q", ntok, nh, hd, dev) if nh else 0, _rows(k, "k", ntok, nkv, hd, dev),
                       _rows(v, "v", ntok, nkv, hd, dev), nh, n_dims, int(neox),
                       cos_sin.data_ptr() if n_dims else None, cos_sin.shape[0] if n_dims else 0,
                       out.data_ptr() if nh else None, _rows(out, "out", ntok, nh, hd, dev) if nh else 0)
    check(lib().lnship16_rope_store_kv_paged(ctypes.byref(kv), ctypes.byref(a), _stream()))
    return out


def attention(q, k_pages, v_pages, page, table, q_start, kv_len, scale, window=0, out=None):
    """Attention of the new tokens q [ntok, n_head, head_dim] float32 over
    their sequences' cells in the pages: those up to each token's own position
    and, with window > 0, no further than window - 1 before it.  Returns out,
    [ntok, n_head, head_dim] float32."""
    import torch
    init()
    ntok, nh = q.shape[0], q.shape[1]
    kv = _kv(k_pages, v_pages, page, table, q_start, kv_len, ntok)
    dev, hd = k_pages.device, kv.head_dim
    if out is None:
        out = torch.empty((ntok, nh, hd), dtype=torch.float32, device=dev)
    q_ld, out_ld = _rows(q, "q", ntok, nh, hd, dev), _rows(out, "out", ntok, nh, hd, dev)
    need = lib().lnship16_attn_paged_work(ctypes.byref(kv), nh)
    if need < 0:
        check(need)
    # (of torch's allocator: the stream's own, a captured graph's own)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    a = PagedAttnArgs(q.data_ptr(), out.data_ptr(), q_ld, out_ld, nh, scale, window,
                      work.data_ptr() if need else None, need)
    check(lib().lnship16_attn_paged(ctypes.byref(kv), ctypes.byref(a), _stream()))
    return out
