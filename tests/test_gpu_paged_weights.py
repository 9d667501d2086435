"""Attention where most of the weight lies on cells of little value, so that the result is the sum of
many small weights: each is off by at most 2^-34 of the row's largest."""
import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import run_attn

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ln():
    import lnship
    import lnship.paged
    lnship.init()
    return lnship


@pytest.mark.parametrize("q_len,cells", [([1], 0), ([90], 0), ([90], 1 << 14), ([260], 1 << 14)])
@pytest.mark.parametrize("sink", [9.0, 12.0, 14.0, 15.25, 17.5, 18.9, 19.25, 20.5, 24.0])
def test_a_cell_without_value_takes_the_weight(ln, q_len, cells, sink):
    """The first cell outweighs each other one by e^sink and its value is zero; the others' are alike in
    sign, so that errors add up.  A weight is a half and the rest of it as a half, of 2^10 times its share
    of the largest: steps of 2^-24, so half a step is 2^-35 of the largest weight.  As much is lost where
    the value's low half (at most the value, times 2^11) meets the weight's copy (times 2^-11), which has
    the same steps.  Everything else is as paged_reference.tolerance() derives it."""
    rng = np.random.default_rng(int(sink * 4))
    page, nkv, hd, n = 16, 2, 64, 300
    k = np.zeros((n, nkv, hd), np.float32)
    v = 1000 * (1 + rng.random((n, nkv, hd)).astype(np.float32))
    k[1:, :, 0] = -1.0
    v[0] = 0.0
    keys, vals = R.store_codes(k), R.store_codes(v)
    table, n_pages = R.tables(rng, [n], page)
    c = R.Cache(n_pages, page, nkv, hd)
    c.put(table[0], np.arange(n), keys, vals)
    q = np.zeros((q_len[0], 4, hd), np.float32)
    q[:, :, 0] = sink + np.arange(4) * 0.11
    got = run_attn(ln, q, c, table, q_len, [n], scale=1.0, cells=cells).cpu().numpy()
    ref, tol = R.attention(q, keys, vals, np.arange(n - q_len[0], n), 1.0)
    tol += 2.0 ** -34 * np.repeat(np.abs(R.value(vals)).sum(0), 2, 0)
    err = np.abs(got - ref)
    print(f"\n[weights] sink {sink} q {q_len} cells {cells}: {(err / tol).max():.3f} of the bound, "
          f"{(err / np.abs(ref)).max():.2e} of the value, {err.max() / R.value(vals).sum(0).max():.2e} of the values' sum",
          flush=True)
    assert (err <= tol).all(), float((err / tol).max())
