"""Pins of Oracle.attention_packed at values that are not finite, without a GPU: which
keys count, and what infinities and NaN do to the rows that see them."""
import numpy as np


def _one(q, k, v, **kw):
    d = len(q)
    o, tol = _one.orc.attention_packed(np.array([q], np.float32), np.array(k, np.float32), np.array(v, np.float32),
                                       np.zeros((1, d)), [(0, 1, 0, len(k))], 1, 1, 1.0, **kw)
    return o[0], tol[0]


def test_what_a_hidden_key_holds_does_not_matter(orc):
    _one.orc = orc
    b = np.array([[-np.inf, 0.0, 0.0, 0.0, 0.0]])  # hides the keys two and more in front of the last one
    for bad in (np.nan, np.inf, -np.inf, 1e30):
        o, tol = _one([1.0, 2.0], [[bad, 0], [0, bad], [1, 1], [1, 1]], [[bad, 1], [1, bad], [2, 3], [4, 5]], bias=b, radius=2)
        assert np.allclose(o, [3, 4], rtol=0, atol=1e-12) and np.all(tol < 2e-4)
    o, tol = _one([1.0, 2.0], [[np.nan, 0]], [[np.nan, 0]], bias=np.full((1, 1), -np.inf), radius=0)
    assert np.all(o == 0) and np.all(tol == 0)


def test_infinite_keys(orc):
    _one.orc = orc
    inf = np.inf
    o, _ = _one([1.0, 0.5], [[-inf, 0], [0, 0], [0, 0]], [[inf, np.nan], [2, 3], [4, 5]])  # a score of -inf: no weight
    assert np.allclose(o, [3, 4], rtol=0, atol=1e-12)
    assert np.all(np.isnan(_one([1.0, 0.5], [[inf, 0], [0, 0]], [[1, 1], [1, 1]])[0]))
    assert np.all(np.isnan(_one([0.0, 0.5], [[inf, 0], [0, 0]], [[1, 1], [1, 1]])[0]))  # 0 * inf
    o, _ = _one([1.0, 0.5], [[inf, 0], [-inf, 0]], [[1, 0], [0, 1]], cap=2.0)  # scores of 2 and -2
    assert np.allclose(o, [1 / (1 + np.exp(-4)), 1 / (1 + np.exp(4))], rtol=0, atol=1e-12)


def test_infinite_values_show_whatever_their_weight(orc):
    _one.orc = orc
    o, tol = _one([1.0, 0.0], [[-3000, 0], [0, 0]], [[np.inf, 1], [1, 2]])
    assert o[0] == np.inf and abs(o[1] - 2) < 1e-12 and np.all(np.isfinite(tol))
    o, _ = _one([1.0, 0.0], [[-3000, 0], [0, 0]], [[np.inf, -np.inf], [-np.inf, 2]])
    assert np.isnan(o[0]) and o[1] == -np.inf


def test_the_largest_value_does_not_lower_the_others_bound(orc):
    """A key of no weight adds nothing to the bound, however large its value."""
    _one.orc = orc
    o, tol = _one([1.0, 0.0], [[-200, 0], [0, 0]], [[1e30, 1e30], [1, 2]])
    assert np.allclose(o, [1, 2], rtol=0, atol=1e-12) and np.all(tol < 2e-4)
