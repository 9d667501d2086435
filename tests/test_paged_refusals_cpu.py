"""What the paged-cache and token-draw entry points refuse, without a GPU: bad shapes and pointers
are refused before any device call (LNSHIP_EINVAL -1, LNSHIP_ERANGE -4), sound arguments get as far as
the device (LNSHIP_ENOINIT -3 where lnship_init was not called)."""
import ctypes

import pytest

import lnship

EINVAL, EDEVICE, ENOINIT, ERANGE = -1, -2, -3, -4
P = 0x10000     # an aligned address that nothing reads


def paged(**kw):
    a = dict(k_pages=P, v_pages=P, n_pages=8, page=16, n_head_kv=2, head_dim=64, table=P, table_ld=4, ntok=3, n_seq=2,
             q_start=P, kv_len=P)
    a.update(kw)
    return lnship.PagedKV(*(a[f[0]] for f in lnship.PagedKV._fields_))


def store(kv=None, **kw):
    a = dict(q=P, k=P, v=P, q_ld=512, k_ld=128, v_ld=128, n_head=8, rope_n_dims=64, neox=0, cos_sin=P, n_pos=64, q_dst=P,
             q_dst_ld=0)
    a.update(kw)
    s = lnship.PagedStoreArgs(*(a[f[0]] for f in lnship.PagedStoreArgs._fields_))
    return lnship.lib().lnship16_rope_store_kv_paged(ctypes.byref(kv or paged()), ctypes.byref(s), None)


def attn(kv=None, **kw):
    a = dict(q=P, dst=P, q_ld=0, dst_ld=0, n_head=8, scale=0.125, window=0, work=P, work_bytes=1 << 40)
    a.update(kw)
    s = lnship.PagedAttnArgs(*(a[f[0]] for f in lnship.PagedAttnArgs._fields_))
    return lnship.lib().lnship16_attn_paged(ctypes.byref(kv or paged()), ctypes.byref(s), None)


def draw(**kw):
    a = dict(logits=P, ld=0, n_rows=2, n_vocab=100, temperature=None, top_k=None, top_p=None, min_p=None, u=P, tokens=P,
             probs=None)
    a.update(kw)
    s = lnship.SampleArgs(*(a[f[0]] for f in lnship.SampleArgs._fields_))
    return lnship.lib().lnship_sample(ctypes.byref(s), None)


@pytest.fixture(autouse=True)
def no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the pointers here are not device memory")


def test_sound_arguments_reach_the_device():
    assert store() in (ENOINIT, EDEVICE) and attn() in (ENOINIT, EDEVICE) and draw() in (ENOINIT, EDEVICE)


BAD_CACHE = [dict(page=8), dict(page=24), dict(page=512), dict(page=0), dict(page=-16), dict(head_dim=0),
             dict(head_dim=12), dict(head_dim=264), dict(head_dim=-8), dict(n_head_kv=0), dict(n_head_kv=-1),
             dict(ntok=-1), dict(n_seq=-1), dict(n_pages=-1), dict(table_ld=-1), dict(k_pages=None),
             dict(v_pages=None), dict(k_pages=P + 8), dict(v_pages=P + 2), dict(q_start=None), dict(kv_len=None),
             dict(table=None)]


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_bad_caches_are_refused(kw):
    assert store(paged(**kw)) == EINVAL and lnship.lib().lnship_last_error()
    assert attn(paged(**kw)) == EINVAL


@pytest.mark.parametrize("kw", [dict(ntok=1 << 24), dict(n_seq=1 << 23), dict(n_head_kv=65536), dict(n_pages=1 << 31),
                                dict(table_ld=1 << 27)], ids=str)
def test_caches_too_large_are_refused(kw):
    wide = dict(k_ld=1 << 40, v_ld=1 << 40)
    assert store(paged(**kw), **wide) == ERANGE and attn(paged(**kw)) == ERANGE


@pytest.mark.parametrize("kw", [dict(n_head=-1), dict(rope_n_dims=-2), dict(rope_n_dims=3), dict(rope_n_dims=66),
                                dict(q_ld=511), dict(k_ld=127), dict(v_ld=127), dict(q_dst_ld=511), dict(n_pos=-1),
                                dict(q=None), dict(k=None), dict(v=None), dict(cos_sin=None), dict(q_dst=None)], ids=str)
def test_bad_stores_are_refused(kw):
    assert store(**kw) == EINVAL


@pytest.mark.parametrize("kw", [dict(n_head=0), dict(n_head=7), dict(n_head=65536), dict(window=-1), dict(q_ld=511),
                                dict(dst_ld=100), dict(q=None), dict(dst=None)], ids=str)
def test_bad_attention_is_refused(kw):
    assert attn(**kw) == EINVAL
    assert lnship.lib().lnship16_attn_paged(None, None, None) == EINVAL


@pytest.mark.parametrize("kw,rc", [(dict(n_rows=-1), EINVAL), (dict(n_vocab=0), EINVAL), (dict(n_vocab=-1), EINVAL),
                                   (dict(ld=99), EINVAL), (dict(logits=None), EINVAL), (dict(u=None), EINVAL),
                                   (dict(tokens=None), EINVAL), (dict(n_vocab=(1 << 19) + 1), ERANGE),
                                   (dict(n_rows=1 << 22), ERANGE)], ids=str)
def test_bad_draws_are_refused(kw, rc):
    assert draw(**kw) == rc
    assert lnship.lib().lnship_sample(None, None) == EINVAL


def test_empty_calls_need_no_pointers():
    none = dict(k_pages=None, v_pages=None, table=None, q_start=None, kv_len=None)
    for e in (dict(ntok=0), dict(n_seq=0)):
        kv = paged(**none, **e)
        assert store(kv, q=None, k=None, v=None, q_dst=None, cos_sin=None) == 0
        assert attn(kv, q=None, dst=None, work=None, work_bytes=0) == 0
    assert draw(n_rows=0, logits=None, u=None, tokens=None) == 0


def test_workspace_sizes():
    L = lnship.lib()
    assert L.lnship16_attn_paged_work(ctypes.byref(paged(page=8)), 8) == EINVAL
    assert L.lnship16_attn_paged_work(ctypes.byref(paged()), 7) == EINVAL


@pytest.mark.parametrize("packer,cls", [("_KV", "PagedKV"), ("_STORE", "PagedStoreArgs"), ("_ATTN", "PagedAttnArgs")])
def test_packed_arguments_are_the_structures(packer, cls):
    import lnship.paged
    cls, packer = getattr(lnship, cls), getattr(lnship.paged, packer)
    n = len(cls._fields_)
    want = [i + 1 + (i << 33) if ctypes.sizeof(t) == 8 else i + 1 for i, (_, t) in enumerate(cls._fields_)]
    a = cls.from_buffer_copy(packer.pack(*want))
    assert packer.size == ctypes.sizeof(cls) and [getattr(a, f[0]) for f in cls._fields_] == want and n == len(want)


def test_tensors_that_are_not_on_the_gpu_are_refused():
    import lnship.paged
    import torch
    k, v = lnship.paged.alloc_pages(4, 16, 2, 64, device="cpu")
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(lnship.LnshipError):
        lnship.paged.attention(torch.zeros(1, 4, 64), k, v, 16, i.view(1, 2), i, i[:1], 0.1)
    with pytest.raises(lnship.LnshipError):
        lnship.sample(torch.zeros(2, 5), torch.zeros(2))
