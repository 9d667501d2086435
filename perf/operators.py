"""The operators of a serving step over a paged cache, as cases that can be timed and compared.

Three operators: the rotation of the queries and keys with the stores into a paged xlns16 cache
(`store`), the attention of each sequence's chunk of new tokens over that cache (`attn`), and the
draw of the next tokens from their logits (`draw`).  With `own` false run() computes them from
elementary torch operations; with `own` true it makes the calls of the framework's package.

Head shapes are those of the two decoder configurations (SmolLM2-135M: 9 query heads on 3 key
heads of 64; Llama 1B: 32 on 8 of 64) and a wider generic one (32 on 8 of 128).  A case's ragged
lengths come from its own numbers (`mix` seeds them), its values from the seed.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
THETA = 10000.0


def listed():
    return [
        # the next token of one user's chat: SmolLM2 heads, one row into the cache
        {"name": "store_token", "kind": "store", "seqs": 1, "q_lo": 1, "q_hi": 1, "past_lo": 300, "past_hi": 300,
         "heads": 9, "kv_heads": 3, "dim": 64, "page": 16, "neox": False, "mix": 1},
        # a decode step of 256 users whose conversations are at different lengths
        {"name": "store_tokens_256", "kind": "store", "seqs": 256, "q_lo": 1, "q_hi": 1, "past_lo": 1, "past_hi": 8000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "neox": True, "mix": 2},
        # prompts of eight users entering the cache, ragged, some behind an earlier turn
        {"name": "store_prompts", "kind": "store", "seqs": 8, "q_lo": 511, "q_hi": 2047, "past_lo": 0, "past_hi": 1500,
         "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "neox": False, "mix": 3},
        # one user's next token, SmolLM2 heads, a short conversation: latency
        {"name": "attn_token", "kind": "attn", "seqs": 1, "q_lo": 1, "q_hi": 1, "past_lo": 300, "past_hi": 300,
         "heads": 9, "kv_heads": 3, "dim": 64, "page": 16, "window": 0, "mix": 4},
        # a decode step of 64 users with ragged conversations
        {"name": "attn_tokens_64", "kind": "attn", "seqs": 64, "q_lo": 1, "q_hi": 1, "past_lo": 100, "past_hi": 8000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "mix": 5},
        # the next token behind one very long document
        {"name": "attn_token_long", "kind": "attn", "seqs": 1, "q_lo": 1, "q_hi": 1, "past_lo": 131071,
         "past_hi": 131071, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "window": 0, "mix": 6},
        # new turns of nine chats at once, odd lengths, SmolLM2 heads
        {"name": "attn_turns", "kind": "attn", "seqs": 9, "q_lo": 5, "q_hi": 301, "past_lo": 0, "past_hi": 1777,
         "heads": 9, "kv_heads": 3, "dim": 64, "page": 16, "window": 0, "mix": 7},
        # one chunk of a long prompt: 4096 new tokens behind 4096 in the cache
        {"name": "attn_chunk", "kind": "attn", "seqs": 1, "q_lo": 4096, "q_hi": 4096, "past_lo": 4096,
         "past_hi": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "mix": 8},
        # two prompts in a layer whose heads see a sliding window of 1000 cells
        {"name": "attn_window", "kind": "attn", "seqs": 2, "q_lo": 1900, "q_hi": 2500, "past_lo": 0, "past_hi": 700,
         "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "window": 1000, "mix": 9},
        # one user's next token out of SmolLM2's vocabulary
        {"name": "draw_token", "kind": "draw", "rows": 1, "vocab": 49152, "mix": 10},
        # a decode step of 61 users, Llama 1B's vocabulary
        {"name": "draw_tokens_61", "kind": "draw", "rows": 61, "vocab": 32000, "mix": 11},
        # a decode step of 256 users, a large vocabulary of odd size
        {"name": "draw_tokens_256", "kind": "draw", "rows": 256, "vocab": 131075, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case: sizes over the ranges of the listed ones, at most the largest listed case's cost."""
    mix = rng.randrange(100, 1 << 20)
    kind = rng.choice(("store", "attn", "attn", "draw"))
    if kind == "draw":
        vocab = _log_int(rng, 1000, 131075)
        return {"kind": kind, "rows": _log_int(rng, 1, 256), "vocab": vocab, "mix": mix}
    heads, kv_heads, dim = rng.choice(((9, 3, 64), (32, 8, 64), (32, 8, 128), (8, 8, 96), (16, 1, 128), (28, 4, 80)))
    page = rng.choice((16, 32, 64, 128))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "mix": mix}
    while True:
        seqs = _log_int(rng, 1, 64)
        q_hi = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        past_hi = _log_int(rng, 1, 131071 if seqs == 1 and q_hi == 1 else 16000)
        # tokens in all, cells in all, and the scores of a batch padded to its longest member
        if seqs * q_hi <= 8192 and seqs * (q_hi + past_hi) <= 300000 and \
                seqs * heads * q_hi * (q_hi + past_hi) <= 32 * 4096 * 8192:
            break
    case.update(seqs=seqs, q_lo=max(1, q_hi // 4), q_hi=q_hi, past_lo=past_hi // 8, past_hi=past_hi)
    if kind == "store":
        case["neox"] = rng.random() < 0.5
    else:
        case["window"] = rng.choice((0, 0, _log_int(rng, 16, 4096)))
    return case


def _lengths(case):
    """The new tokens and the cells (new ones among them) of each sequence."""
    r = random.Random(case["mix"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    return q, [n + r.randint(case["past_lo"], case["past_hi"]) for n in q]


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _random_codes(shape, g):
    """xlns16 codes of normally distributed values."""
    n = math.prod(shape)
    out = torch.empty(n, dtype=torch.int16, device=DEV)
    for i in range(0, n, 1 << 26):
        x = torch.randn(min(1 << 26, n - i), generator=g, device=DEV)
        c = (x.abs().clamp_min(1e-6).log2() * 128).to(torch.int32) + 0x4000
        out[i:i + x.numel()] = torch.where(x < 0, c - 0x8000, c).to(torch.int16)
    return out.view(shape)


def _prepare_paged(case, seed):
    g = _gen(seed)
    q_len, kv_len = _lengths(case)
    S, page, nh, nkv, hd = case["seqs"], case["page"], case["heads"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in kv_len]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV)[:sum(need)].to(torch.int32)
    table = torch.full((S, max(need)), -1, dtype=torch.int32)
    rows = torch.repeat_interleave(torch.arange(S), torch.tensor(need))
    cols = torch.cat([torch.arange(n) for n in need])
    table[rows, cols] = order.cpu()
    start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
    st = {"case": case, "ntok": int(start[-1]), "max_q": max(q_len), "max_kv": max(kv_len),
          "table": table.to(DEV), "q_start": torch.from_numpy(start).to(DEV),
          "kv_len": torch.tensor(kv_len, dtype=torch.int32, device=DEV)}
    T = st["ntok"]
    if case["kind"] == "store":
        # the rows of a fused q|k|v product
        st["qkv"] = torch.randn((T, (nh + 2 * nkv) * hd), generator=g, device=DEV)
        t = torch.arange(max(kv_len), dtype=torch.float64)[:, None]
        a = t * THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
        st["cos_sin"] = torch.stack((a.cos(), a.sin()), -1).float().to(DEV)
        st["q_out"] = torch.empty((T, nh, hd), device=DEV)
    else:
        # queries of a trained model lean on few cells: scores of standard deviation 2
        st["q"] = torch.randn((T, nh, hd), generator=g, device=DEV) * 2
        st["out"] = torch.empty((T, nh, hd), device=DEV)
    st["k"] = _random_codes((n_pages, nkv, page * hd), g)
    st["v"] = _random_codes((n_pages, nkv, page * hd), g)
    return st


def _prepare_draw(case, seed):
    g = _gen(seed)
    R, V = case["rows"], case["vocab"]
    x = torch.randn((R, V), generator=g, device=DEV) * 2.5
    # a few likely tokens stand out, as a trained model's do
    hot = torch.randint(0, V, (R, 40), generator=g, device=DEV)
    x.scatter_add_(1, hot, torch.rand((R, 40), generator=g, device=DEV) * 9)
    # each user's own settings: some draw from all tokens, some take the likeliest
    c = torch.rand((4, R), generator=g, device=DEV)
    temp = torch.where(c[0] < 0.1, torch.zeros_like(c[0]), 0.5 + c[0])
    top_k = torch.where(c[1] < 0.4, torch.zeros_like(c[1]), 1 + c[1] * 200).to(torch.int32)
    top_p = torch.where(c[2] < 0.3, torch.ones_like(c[2]), 0.5 + 0.5 * c[2])
    min_p = torch.where(c[3] < 0.6, torch.zeros_like(c[3]), 0.1 * c[3])
    return {"case": case, "logits": x, "temperature": temp, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "u": torch.rand(R, generator=g, device=DEV),
            "tokens": torch.empty(R, dtype=torch.int32, device=DEV), "probs": torch.empty(R, device=DEV)}


def prepare(case, seed):
    return (_prepare_draw if case["kind"] == "draw" else _prepare_paged)(case, seed)


# ---- the framework's calls -----------------------------------------------------------------------

def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xlns-ggml-backend_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import lnship
    import lnship.paged
    return lnship


def _own(st):
    ln, case = _package(), st["case"]
    if case["kind"] == "draw":
        return ln.sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                         min_p=st["min_p"], out=(st["tokens"], st["probs"]))
    nh, nkv, hd, T = case["heads"], case["kv_heads"], case["dim"], st["ntok"]
    if case["kind"] == "store":
        qkv = st["qkv"].view(T, nh + 2 * nkv, hd)
        ln.paged.rope_store_kv(qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:], st["k"], st["v"], case["page"],
                               st["table"], st["q_start"], st["kv_len"], st["cos_sin"], neox=case["neox"],
                               out=st["q_out"])
        return {"q": st["q_out"], "k": st["k"], "v": st["v"]}
    return ln.paged.attention(st["q"], st["k"], st["v"], case["page"], st["table"], st["q_start"], st["kv_len"],
                              scale=1.0 / math.sqrt(hd), window=case["window"], out=st["out"])


# ---- the plain forms -----------------------------------------------------------------------------

def _encode(x):
    """The xlns16 codes of F32 values: 128 log2|x| truncated toward zero (of x's upper 8 mantissa
    bits), offset by 0x4000, under the sign bit; 0 for zero."""
    x = (x.contiguous().view(torch.int32) & -0x8000).view(torch.float32)
    log = (x.abs().double().log2() * 128).trunc()
    code = torch.where(x == 0, 0, log + 0x4000).to(torch.int32)
    return torch.where(x < 0, code | 0x8000, code)


def _decode(code):
    """The F32 values of xlns16 codes."""
    log = code.to(torch.int32) & 0x7fff
    x = torch.where(log == 0, 0.0, torch.exp2(log.float() * (1 / 128) - 128))
    return torch.where((code & 0x8000) != 0, -x, x)


def _mul(a, b):
    log = ((a & 0x7fff) + (b & 0x7fff) - 0x4000).clamp(0, 0x7fff)
    return ((a ^ b) & 0x8000) | log


def _add(a, b):
    """The xlns16 sum: the larger log plus the Gaussian log of the distance, in steps of 1/128 binade."""
    la, lb = a & 0x7fff, b & 0x7fff
    d = (la - lb).abs()
    opposite = ((a ^ b) & 0x8000) != 0
    ratio = torch.exp2(d.double() / 128)
    adjust = -d + (torch.where(opposite, ratio - 1, ratio + 1).log2() * 128 + 0.5).clamp(-1e6, 1e6).to(torch.int32)
    adjust = torch.where(d > 1280, 0, adjust)
    log = (torch.maximum(la, lb) + adjust).clamp(0, 0x7fff)
    return torch.where(opposite & (d == 0), 0, (torch.where(la > lb, a, b) & 0x8000) | log)


def _rotate(x, cs, neox):
    """The rotated codes of x [T, heads, dim] by the (cos, sin) pairs cs [T, dim / 2, 2]."""
    T, n, hd = x.shape
    code = _encode(x)
    c, s = _encode(cs[:, None, :, 0]), _encode(cs[:, None, :, 1])
    a, b = (code[..., :hd // 2], code[..., hd // 2:]) if neox else (code[..., 0::2], code[..., 1::2])
    r0 = _add(_mul(a, c), _mul(b, s) ^ 0x8000)
    r1 = _add(_mul(a, s), _mul(b, c))
    return torch.cat((r0, r1), -1) if neox else torch.stack((r0, r1), -1).reshape(T, n, hd)


def _rows(st):
    """Each token's sequence and position."""
    t = torch.arange(st["ntok"], device=DEV)
    seq = torch.bucketize(t, st["q_start"][1:].long(), right=True)
    return seq, st["kv_len"][seq] - st["q_start"][seq + 1] + t


def _plain_store(st):
    case = st["case"]
    nh, nkv, hd, page, T = case["heads"], case["kv_heads"], case["dim"], case["page"], st["ntok"]
    seq, pos = _rows(st)
    x = st["qkv"].view(T, nh + 2 * nkv, hd)
    rotated = _decode(_rotate(x[:, :nh + nkv], st["cos_sin"][pos], case["neox"]))
    k, v = (_encode(y.half().float()).to(torch.int16) for y in (rotated[:, nh:], x[:, nh + nkv:]))
    at = st["table"][seq, pos // page].long(), pos % page
    # a page's keys: eight dimensions of a cell together; its values: eight cells of a dimension
    st["k"].view(-1, nkv, hd // 8, page, 8).permute(0, 3, 1, 2, 4)[at] = k.view(T, nkv, hd // 8, 8)
    st["v"].view(-1, nkv, page // 8, hd, 8).permute(0, 2, 4, 1, 3)[at[0], at[1] // 8, at[1] % 8] = v
    st["q_out"].copy_(rotated[:, :nh])
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _cells(st):
    """Keys and values of every sequence as codes, [S, kv head, cell, dim], padded to the longest."""
    case = st["case"]
    nkv, hd, page = case["kv_heads"], case["dim"], case["page"]
    table = st["table"].clamp_min(0).long()
    S, P = table.shape
    k = st["k"].view(-1, nkv, hd // 8, page, 8)[table].permute(0, 2, 1, 4, 3, 5).reshape(S, nkv, P * page, hd)
    v = st["v"].view(-1, nkv, page // 8, hd, 8)[table].permute(0, 2, 1, 3, 5, 4).reshape(S, nkv, P * page, hd)
    return k, v


def _plain_attn(st):
    case = st["case"]
    nh, nkv, hd, S, Q = case["heads"], case["kv_heads"], case["dim"], case["seqs"], st["max_q"]
    k, v = (_decode(c) for c in _cells(st))
    J = k.shape[2]
    seq, pos = _rows(st)
    i = torch.arange(st["ntok"], device=DEV) - st["q_start"][seq]
    # the chunks padded to the longest: [S, kv head, heads of the group, Q, dim]
    q = torch.zeros((S, Q, nh, hd), device=DEV)
    q[seq, i] = st["q"]
    q = q.view(S, Q, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(S, nkv, -1, hd)
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    at = torch.full((S, Q), -1, device=DEV, dtype=pos.dtype)
    at[seq, i] = pos
    j = torch.arange(J, device=DEV)
    seen = j <= at[:, :, None]
    if case["window"]:
        seen &= j > at[:, :, None] - case["window"]
    s = s.view(S, nkv, nh // nkv, Q, J).masked_fill_(~seen[:, None, None], -math.inf)
    s = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(S, nkv, -1, J), v).view(S, nkv, nh // nkv, Q, hd) / total.clamp_min(1e-30)
    st["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(S, Q, nh, hd)[seq, i])
    return st["out"]


def _plain_draw(st):
    x = st["logits"]
    V = x.shape[1]
    # 64 bits: a token is kept, or drawn, by comparing sums of up to all weights
    order = x.sort(dim=1, descending=True, stable=True)
    T = st["temperature"].double()[:, None]
    greedy = T <= 0
    xs = order.values.double()
    w = ((xs - xs[:, :1]) / torch.where(greedy, 1.0, T)).exp()
    rank = torch.arange(V, device=DEV)
    k = torch.where(st["top_k"] > 0, st["top_k"], V)[:, None]
    w = torch.where(rank < torch.where(greedy, 1, k), w, 0.0)
    before = w.cumsum(1) - w
    top_p, min_p = st["top_p"].double()[:, None], st["min_p"].double()[:, None]
    keep = (top_p >= 1) | (before < top_p * w.sum(1, keepdim=True)) | (rank == 0)
    keep &= (w >= min_p) | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, order.indices, torch.where(keep, w, 0.0))
    c = w.cumsum(1)
    token = (c <= st["u"].double()[:, None] * c[:, -1:]).sum(1, keepdim=True).clamp_max(V - 1)
    st["tokens"].copy_(token[:, 0])
    st["probs"].copy_((w.gather(1, token) / c[:, -1:])[:, 0])
    return st["tokens"], st["probs"]


def run(st):
    if own:
        return _own(st)
    return {"store": _plain_store, "attn": _plain_attn, "draw": _plain_draw}[st["case"]["kind"]](st)


def work(case):
    if case["kind"] == "draw":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    q, kv = _lengths(case)
    T = sum(q)
    if case["kind"] == "store":
        # q, k, v and a row of (cos, sin) in; q in 32 bits, k and v in 16 out; a pair is four products and two sums
        return {"bytes": T * hd * (4 * (nh + 2 * nkv) + 4 + 4 * nh + 2 * 2 * nkv), "flops": T * (nh + nkv) * hd * 3}
    w = case["window"] or 1 << 40
    seen = sum(min(p + 1, w) for n, m in zip(q, kv) for p in range(m - n, m))
    cells = sum(m - max(0, m - n - w + 1) for n, m in zip(q, kv))
    return {"bytes": 8 * T * nh * hd + 4 * cells * nkv * hd, "flops": 4 * hd * nh * seen}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _value(code):
    """The real numbers that xlns16 codes stand for, in 64 bits."""
    c = code.long()
    size = torch.pow(2.0, ((c & 0x7fff) - 0x4000).double() / 128)
    return size * ((c & 0x7fff) != 0) * torch.where(c & 0x8000 != 0, -1.0, 1.0).double()


def _exact_attn(st):
    case = st["case"]
    nh, nkv, hd, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros((st["ntok"], nh, hd), dtype=torch.float64, device=DEV)
    start, kv = st["q_start"].tolist(), st["kv_len"].tolist()
    for s in range(case["seqs"]):
        n = kv[s]
        ids = st["table"][s, :-(-n // page)].long()
        for g in range(nkv):
            key = _value(st["k"][ids, g].view(-1, hd // 8, page, 8).transpose(1, 2).reshape(-1, hd)[:n])
            val = _value(st["v"][ids, g].view(-1, page // 8, hd, 8).transpose(2, 3).reshape(-1, hd)[:n])
            for r in range(start[s], start[s + 1], 1024):
                e = min(start[s + 1], r + 1024)
                pos = n - start[s + 1] + torch.arange(r, e, device=DEV)
                j = torch.arange(n, device=DEV)
                hidden = j[None] > pos[:, None]
                if case["window"]:
                    hidden |= j[None] <= pos[:, None] - case["window"]
                for h in range(g * (nh // nkv), (g + 1) * (nh // nkv)):
                    z = st["q"][r:e, h].double() @ key.T / math.sqrt(hd)
                    out[r:e, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ val
    return out


def _exact_store(st):
    """The rotated queries: the pairs' products and sums on logs in steps of 1/128 binade, in numpy."""
    case = st["case"]
    nh, hd, T = case["heads"], case["dim"], st["ntok"]
    if T * nh * hd > 32 << 20:
        return None
    q_len, kv_len = _lengths(case)
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(q_len, kv_len)])
    x = st["qkv"].cpu().numpy().reshape(T, -1, hd)[:, :nh]
    cs = st["cos_sin"].cpu().numpy()[pos][:, None]

    def log(y):   # (steps, sign) of F32 values; the conversion reads the upper 8 mantissa bits
        y = (y.view(np.uint32) & np.uint32(0xffff8000)).view(np.float32).astype(np.float64)
        with np.errstate(divide="ignore"):
            return np.where(y == 0, -np.inf, np.trunc(128 * np.log2(np.abs(y)))), np.sign(y)

    def plus(a, b):
        (la, sa), (lb, sb) = a, b
        hi, d = np.maximum(la, lb), np.abs(la - lb)
        with np.errstate(divide="ignore", invalid="ignore"):
            # the rounded log of 2^(d/128) +- 1, cut toward zero as a C cast does
            z = np.trunc(128 * np.log2(np.exp2(np.minimum(d, 2000) / 128) + np.where(sa == sb, 1, -1)) + 0.5) - d
        z = np.where(d > 1280, 0, z)
        return np.where((d == 0) & (sa != sb), -np.inf, hi + z), np.where(la > lb, sa, sb)

    a, b = (x[..., :hd // 2], x[..., hd // 2:]) if case["neox"] else (x[..., ::2], x[..., 1::2])
    (a, sa), (b, sb) = log(np.ascontiguousarray(a)), log(np.ascontiguousarray(b))
    (c, sc), (s, ss) = log(np.ascontiguousarray(cs[..., 0])), log(np.ascontiguousarray(cs[..., 1]))
    r = plus((a + c, sa * sc), (b + s, -sb * ss)), plus((a + s, sa * ss), (b + c, sb * sc))
    r = [np.where(np.isinf(l), 0, sg * np.exp2(np.maximum(l, -16384) / 128)) for l, sg in r]
    q = np.concatenate(r, -1) if case["neox"] else np.stack(r, -1).reshape(T, nh, hd)
    return {"q": q, "k": None, "v": None}


def _exact_draw(st):
    x = st["logits"].cpu().numpy().astype(np.float64)
    T, k, tp, mp, u = (st[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    tokens, probs = np.zeros(len(x), np.int32), np.ones(len(x))
    for r, row in enumerate(x):
        if T[r] <= 0:
            tokens[r] = row.argmax()
            continue
        best = np.argsort(-row, kind="stable")
        if k[r] > 0:
            best = best[:int(k[r])]
        w = np.exp((row[best] - row[best[0]]) / T[r])
        n = len(w)
        if tp[r] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), tp[r] * w.sum(), side="left"))
        n = max(1, min(n, int((w >= mp[r]).sum())))
        chosen = np.sort(best[:n])
        w = np.exp((row[chosen] - row[best[0]]) / T[r])
        c = np.cumsum(w)
        at = min(int(np.searchsorted(c, u[r] * c[-1], side="right")), len(c) - 1)
        tokens[r], probs[r] = chosen[at], w[at] / c[-1]
    return tokens, probs


def exact(case, seed):
    return {"store": _exact_store, "attn": _exact_attn, "draw": _exact_draw}[case["kind"]](prepare(case, seed))
