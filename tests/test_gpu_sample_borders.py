"""Token draws that one histogram does not resolve, with a min_p at or above the largest token's own
weight: the first token by rank is kept always, and every row's token and probability are written."""
import numpy as np
import pytest

from test_gpu_sample import check, dev

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ln():
    import lnship
    lnship.init()
    return lnship


def draws(ln, x, u, T=None, k=None, p=None, m=None):
    """The draw into outputs that hold what no draw gives."""
    rows = len(x)
    out = (torch.full((rows,), -77, dtype=torch.int32, device="cuda"), torch.full((rows,), -7.0, device="cuda"))
    ln.sample(dev(x, np.float32), dev(u, np.float32), dev(T, np.float32), dev(k, np.int32), dev(p, np.float32),
              dev(m, np.float32), out=out)
    return out[0].cpu().numpy(), out[1].cpu().numpy()


@pytest.mark.parametrize("vocab", [2500, 40000])
@pytest.mark.parametrize("min_p", [0.25, 0.99999994, 1.0, 1.0000001, 5.0, float("inf")])
@pytest.mark.parametrize("what", ["large top_k", "cold", "infinitely hot", "all alike", "ties at the top", "tied border"])
def test_min_p_up_to_the_largest_weight(ln, what, min_p, vocab):
    print(f"\n[draw] {what} min_p {min_p} vocab {vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    rows = 6
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    x[:, 7] = 9.0                     # the largest, alone
    u = np.array([0.0, 0.1, 0.4, 0.5, 0.8, 0.9999999])
    m = np.full(rows, min_p)
    T = k = p = None
    if what == "large top_k":
        k = np.full(rows, 2000)
    elif what == "cold":
        T = np.full(rows, 1e-6)
    elif what == "infinitely hot":
        T = np.full(rows, np.inf)
    elif what == "all alike":
        x[:] = -3.0
        p = np.array([0.0, 0.3, 0.5, 0.9, 0.999, 0.9999999])
    elif what == "ties at the top":
        x[:, 5:2400:3] = 9.0
        k = np.full(rows, 1500)
    else:
        x = np.round(x).astype(np.float32)
        p = np.array([0.0, 0.3, 0.5, 0.9, 0.999, 0.9999999])
    check(draws(ln, x, u, T, k, p, m), x, u, T, k, p, m)


@pytest.mark.parametrize("vocab", [100, 30000, 60000])
def test_a_min_p_above_one_leaves_the_first_token(ln, vocab):
    """Of equal largest logits too, whichever limits stand beside it."""
    rng = np.random.default_rng(vocab)
    rows = 5
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    first = np.array([0, 3, 50, 98, 99])
    for r, f in enumerate(first):
        x[r, f:] = 8.0
    u = np.full(rows, 0.75)
    for kw in ({}, {"T": 0.7}, {"k": 40}, {"k": 5000}, {"p": 0.9}, {"k": 40, "p": 0.9}):
        kw = {n: np.full(rows, y) for n, y in kw.items()}
        for m in (1.5, float("inf")):
            tok, prob = draws(ln, x, u, **kw, m=np.full(rows, m))
            assert np.array_equal(tok, first) and (prob == 1.0).all(), (kw, m)


@pytest.mark.parametrize("vocab", [262145, (1 << 19) - 1, 1 << 19])
@pytest.mark.parametrize("kind", ["smooth", "flat", "alike", "two levels"])
def test_the_largest_vocabularies(ln, vocab, kind):
    """Up to 512 segments, the fewest bits of a bin's weight and its sums' largest."""
    print(f"\n[draw] {vocab} {kind}", flush=True)
    rng = np.random.default_rng(vocab)
    rows = 10
    x = rng.standard_normal((rows, vocab))
    x = {"smooth": x * 2.5, "flat": x * 0.01, "alike": x * 0 - 3, "two levels": np.where(x > 2, 6.0, 0.0) + x * 1e-4}[kind]
    x = x.astype(np.float32)
    u = np.concatenate([[0.0, 0.9999999], rng.random(rows - 2)])
    p = np.concatenate([[1e-7, 0.9999999, 1.0], rng.random(rows - 3)])
    m = np.where(np.arange(rows) % 4 == 3, 0.02, 0.0)
    k = np.where(np.arange(rows) % 3 == 0, 50, 0)
    check(draws(ln, x, u, None, None, p, m), x, u, None, None, p, m)
    check(draws(ln, x, u, None, k, p, m), x, u, None, k, p, m)
    check(draws(ln, x, u), x, u, None, None, None, None)


def test_a_larger_vocabulary_is_refused(ln):
    with pytest.raises(ln.LnshipError, match="too large"):
        ln.sample(torch.zeros((1, (1 << 19) + 1), device="cuda"), torch.zeros(1, device="cuda"))


@pytest.mark.parametrize("vocab", [40000, 131075])
@pytest.mark.parametrize("first", [-np.inf, np.nan, -300.0, 300.0])
def test_rows_whose_first_logits_are_unlike_the_rest(ln, vocab, first):
    """A long row's bins are counted from the largest of its first 16384 logits; here none of those is a
    number, or all lie far from the rest."""
    rng = np.random.default_rng(vocab)
    rows = 8
    x = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    x[:, :17000] = first
    x[::2, 123::5000] = first        # in the rest too
    u = rng.random(rows)
    for kw in ({"p": 0.9}, {"k": 40}, {"k": 40, "p": 0.7}, {"p": 0.99, "m": 0.01}, {"k": 3000}):
        a = [np.full(rows, kw[n]) if n in kw else None for n in ("T", "k", "p", "m")]
        check(draws(ln, x, u, *a), x, u, *a)
