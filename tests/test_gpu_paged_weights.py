"""Attention where most of the weight lies on cells of little value, so that the result is the sum of
many small weights: each keeps its bits relative to the row's largest."""
import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import dev, run_attn

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ln():
    import lnship
    import lnship.paged
    lnship.init()
    return lnship


@pytest.mark.parametrize("q_len,cells", [([1], 0), ([90], 0), ([90], 1 << 14), ([260], 1 << 14)])
@pytest.mark.parametrize("sink", [14.0, 15.25, 17.5, 18.9, 19.25, 20.5])
def test_a_cell_without_value_takes_the_weight(ln, q_len, cells, sink):
    """The first cell outweighs each other one by e^sink and its value is zero.  A weight is a pair of
    halves in steps of 2^-24 of 2^-13 of the row's largest: half a step is 2^-38 of that, and as much
    again is lost where the value's low half meets the weight's copy, which has the same steps.
    paged_reference.tolerance() holds the one; the other is added."""
    rng = np.random.default_rng(int(sink * 4))
    page, nkv, hd, n = 16, 2, 64, 300
    k = np.zeros((n, nkv, hd), np.float32)
    v = rng.standard_normal((n, nkv, hd)).astype(np.float32) * 1000
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
    tol += 2.0 ** -38 * np.repeat(np.abs(R.value(vals)).sum(0), 2, 0)
    err = np.abs(got - ref)
    assert (err <= tol).all(), float((err / tol).max())
