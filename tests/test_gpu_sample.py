"""The token draw on the GPU against a 64-bit form: temperature, top-k, top-p and min-p with ties at
their borders, infinities, NaN and empty rows, odd vocabularies and strides, graphs.

A weight is off by at most 2^-32 of itself (its exponent by 2^-33, its power by 2^-39) and half a unit
of 2^-40, so a share's border by 2^-31 and n 2^-40; a token may differ from the 64-bit form's only where
u lies that near a border.  A probability is rounded to 24 bits besides."""
import numpy as np
import pytest

import paged_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ln():
    import lnship
    lnship.init()
    return lnship


def dev(a, t):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=t)).cuda() if a is not None else None


def run(ln, x, u, T=None, k=None, p=None, m=None, **kw):
    t, pr = ln.sample(x if isinstance(x, torch.Tensor) else dev(x, np.float32), dev(u, np.float32), dev(T, np.float32),
                      dev(k, np.int32), dev(p, np.float32), dev(m, np.float32), **kw)
    return t.cpu().numpy(), pr.cpu().numpy()


def check(got, x, u, T, k, p, m):
    tok, prob = got
    n = x.shape[1]
    eps = 2.0 ** -31 + n * 2.0 ** -40
    for r in range(len(x)):
        one = lambda a, d: float(np.float32(a[r])) if a is not None else d
        want, wp, near = R.draw(x[r], one(T, 1.0), int(one(k, 0)), one(p, 1.0), one(m, 0.0), float(np.float32(u[r])))
        if near > eps:
            assert tok[r] == want, (r, tok[r], want, near)
            assert abs(prob[r] - wp) <= (2 * eps + 2.0 ** -24) * wp + 2.0 ** -40, (r, prob[r], wp)


def settings(rng, rows):
    T = np.where(rng.random(rows) < 0.15, 0.0, 0.3 + rng.random(rows) * 1.5)
    k = np.where(rng.random(rows) < 0.4, 0, rng.integers(1, 100, rows))
    p = np.where(rng.random(rows) < 0.4, 1.0, rng.random(rows))
    m = np.where(rng.random(rows) < 0.5, 0.0, rng.random(rows) * 0.2)
    return T, k, p, m


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1025, 4096, 5001, 32000, 49152, 70001, 131075])
@pytest.mark.parametrize("rows", [1, 7])
def test_draws_equal_64_bits(ln, vocab, rows):
    print(f"\n[draw] {rows} x {vocab}", flush=True)
    rng = np.random.default_rng(vocab + rows)
    for spread in (0.5, 3.0, 12.0):
        x = (rng.standard_normal((rows, vocab)) * spread).astype(np.float32)
        u = rng.random(rows)
        T, k, p, m = settings(rng, rows)
        check(run(ln, x, u, T, k, p, m), x, u, T, k, p, m)
        check(run(ln, x, u), x, u, None, None, None, None)


@pytest.mark.parametrize("vocab", [40, 3000, 60000])
def test_ties_at_every_border(ln, vocab):
    """Logits on a coarse grid: each limit falls among equal ones, of which the first are kept."""
    rng = np.random.default_rng(vocab)
    rows = 64
    x = np.round(rng.standard_normal((rows, vocab)) * 2).astype(np.float32) / 2
    u = rng.random(rows)
    T, k, p, m = settings(rng, rows)
    k = np.where(rng.random(rows) < 0.5, rng.integers(1, vocab + 5, rows), k)
    check(run(ln, x, u, T, k, p, m), x, u, T, k, p, m)
    x[:] = -3.0                                   # all alike
    check(run(ln, x, u, T, k, p, m), x, u, T, k, p, m)


@pytest.mark.parametrize("vocab", [5001, 131075])
@pytest.mark.parametrize("kind", ["smooth", "16 bits", "flat", "tail", "two levels"])
def test_top_p_alone(ln, vocab, kind):
    """Borders anywhere in the sum: among crowded tokens, between far levels, in the tail."""
    rng = np.random.default_rng(vocab)
    rows = 24
    x = rng.standard_normal((rows, vocab))
    x = {"smooth": x * 2.5, "16 bits": x * 8, "flat": x * 0.01, "tail": -4 * np.log(np.abs(x) + 1e-3),
         "two levels": np.where(x > 2, 6.0, 0.0) + x * 1e-4}[kind].astype(np.float32)
    if kind == "16 bits":
        x = (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
    p = np.concatenate([[1e-7, 0.01, 0.9999, 0.99999, 0.9999999], rng.random(rows - 5)])
    m = np.where(np.arange(rows) % 3 == 0, 0.02, 0.0)
    u = rng.random(rows)
    u[::4] = 0.9999999
    check(run(ln, x, u, None, None, p, m), x, u, None, None, p, m)


def test_overlapping_rows_are_refused(ln):
    x = torch.zeros((1, 50), device="cuda")
    u = torch.zeros(3, device="cuda")
    with pytest.raises(ln.LnshipError, match="overlap"):
        ln.sample(x.expand(3, 50), u)
    with pytest.raises(ln.LnshipError, match="overlap"):
        ln.sample(torch.zeros(60, device="cuda").unfold(0, 50, 5), u)


def test_top_k_of_more_than_weigh_anything(ln):
    """Fewer tokens within reach of the largest than top_k: top_p still cuts them."""
    x = np.full((6, 3000), -1e4, np.float32)
    x[:, 70:75] = [3.0, 2.0, 2.5, 1.0, 0.0]
    u, k, p = np.array([0.1, 0.5, 0.7, 0.9, 0.99, 0.999]), np.full(6, 50), np.array([0.5, 0.7, 0.8, 0.9, 0.3, 0.97])
    check(run(ln, x, u, None, k, p), x, u, None, k, p, None)


@pytest.mark.parametrize("vocab", [33, 50000])
def test_limits_at_their_ends(ln, vocab):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, vocab)).astype(np.float32)
    best = int(x.argmax())
    for kw in ({"k": [1]}, {"p": [0.0]}, {"p": [-1.0]}, {"m": [1.0]}, {"m": [5.0]}, {"T": [0.0]}, {"T": [-1.0]},
               {"T": [1e-30]}, {"T": [float("nan")]}):
        for u in (0.0, 0.5, 0.99999994):
            tok, prob = run(ln, x, [u], **kw)
            assert tok[0] == best and prob[0] == 1.0, (kw, u)
    for kw in ({"k": [0]}, {"k": [-5]}, {"k": [vocab]}, {"k": [1 << 30]}, {"p": [1.0]}, {"p": [2.0]},
               {"p": [float("nan")]}, {"m": [0.0]}, {"m": [-1.0]}, {"m": [float("nan")]}):
        u = [0.37]
        assert np.array_equal(run(ln, x, u, **kw)[0], run(ln, x, u)[0]), kw
    # u at its ends: the first and the last token; outside [0, 1) the nearer end
    assert [int(run(ln, x, [u])[0][0]) for u in (0.0, -3.0, float("nan"))] == [0, 0, 0]
    assert [int(run(ln, x, [u])[0][0]) for u in (1.0, 7.0)] == [vocab - 1] * 2
    # an infinite temperature: all alike
    tok, prob = run(ln, x, [0.5], T=[float("inf")])
    assert tok[0] == int(0.5 * vocab) and abs(prob[0] * vocab - 1) < 1e-6


@pytest.mark.parametrize("vocab", [50, 40000])
def test_infinities_nan_and_empty_rows(ln, vocab):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((8, vocab)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, 7] = np.nan
    x[3, :] = -np.inf
    x[3, 11] = -1e38                              # the only number
    x[4, ::2] = -np.inf
    x[5, ::3] = np.nan
    x[6, 5] = x[6, 9] = np.inf
    x[7, 3] = 3e38
    u = np.full(8, 0.6)
    for kw in ({}, {"T": np.full(8, 0.7), "k": np.full(8, 5), "p": np.full(8, 0.8), "m": np.full(8, 0.01)},
               {"T": np.zeros(8)}, {"k": np.full(8, vocab - 1)}):
        tok, prob = run(ln, x, u, **kw)
        assert tok[0] == tok[1] == tok[2] == -1 and (prob[:3] == 0).all()
        assert tok[3] == 11 and prob[3] == 1
        assert tok[4] % 2 == 1 and tok[5] % 3 != 0
        assert tok[6] == (5 if "T" in kw and kw["T"][0] == 0 else 9)
        assert tok[7] == 3
        check((tok[3:6], prob[3:6]), x[3:6], u[3:6], *(kw.get(n)[3:6] if n in kw else None for n in ("T", "k", "p", "m")))


def test_strided_rows_and_given_outputs(ln):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, 777)).astype(np.float32)
    buf = torch.full((5, 1001), float("inf"), device="cuda")
    buf[:, 3:780] = dev(x, np.float32)
    u = rng.random(5)
    out = (torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty(5, device="cuda"))
    got = run(ln, buf[:, 3:780], u, out=out)
    check(got, x, u, None, None, None, None)
    assert np.array_equal(out[0].cpu().numpy(), got[0])


def test_draws_follow_their_distribution(ln):
    """Evenly spaced u over one row draw every token as often as it weighs."""
    rng = np.random.default_rng(4)
    n, rows = 300, 4000
    x = np.repeat((rng.standard_normal((1, n)) * 2).astype(np.float32), rows, 0)
    u = (np.arange(rows) + 0.5) / rows
    tok, prob = run(ln, x, u, T=np.full(rows, 0.8), k=np.full(rows, 50), p=np.full(rows, 0.9))
    order, w = R.kept(x[0], np.float64(np.float32(0.8)), 50, np.float64(np.float32(0.9)), 0)
    got = np.bincount(tok, minlength=n) / rows
    want = np.zeros(n)
    want[order] = w / w.sum()
    assert np.abs(got - want).max() <= 1.0 / rows + 1e-6 and (np.diff(tok) >= 0).all()


def test_the_same_draw_twice_and_replayed(ln):
    rng = np.random.default_rng(5)
    x = dev(rng.standard_normal((9, 40001)) * 2, np.float32)
    u, T = dev(rng.random(9), np.float32), dev(np.full(9, 0.9), np.float32)
    p = dev(np.full(9, 0.95), np.float32)
    want = ln.sample(x, u, T, top_p=p)
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            got = ln.sample(x, u, T, top_p=p)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        x.copy_(dev(rng.standard_normal((9, 40001)) * 2, np.float32))
        u.copy_(dev(rng.random(9), np.float32))
        g.replay()
        have = [t.clone() for t in got]
        if i % 2:
            torch.cuda.synchronize()
        want = ln.sample(x, u, T, top_p=p)
        assert torch.equal(have[0], want[0]) and torch.equal(have[1], want[1])
