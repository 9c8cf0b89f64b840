"""Pins of the oracles of packed-sequence attention and of low-rank adapters
(Oracle.attention_packed, Oracle.lora), without a GPU: against Oracle.attention
(itself pinned to the reference) sequence by sequence, against the plain linear
layer, closed forms of each mask, and planted mistakes."""
import numpy as np
import pytest


def _packed(orc, n, heads, kv, d, seed):
    """Sequences of n rows each, packed, with the same queries' and keys' spans."""
    T = sum(n)
    q, k, v = orc.randn((T, heads * d), seed), orc.randn((T, kv * d), seed + 1), orc.randn((T, kv * d), seed + 2)
    first = np.concatenate(([0], np.cumsum(n)[:-1]))
    return q, k, v, np.array([(f, m, f, m) for f, m in zip(first, n)], np.int32)


@pytest.mark.parametrize("causal", [False, True])
def test_sequences_equal_their_own_attention(orc, causal):
    heads, kv, d, n = 4, 2, 16, [3, 1, 0, 11]
    q, k, v, spans = _packed(orc, n, heads, kv, d, 40)
    scale = float(np.float32(1) / np.sqrt(np.float32(d)))
    got, _ = orc.attention_packed(q, k, v, np.zeros_like(q), spans, heads, kv, scale, causal)
    for f, m, _, _ in spans:
        if m:
            want = orc.attention(q[None, f:f + m], k[None, f:f + m], v[None, f:f + m], heads, causal, kv)
            assert np.max(np.abs(got[f:f + m] - want[0])) <= 2.0 ** -22


def _pin_masks(orc):
    """Equal keys give the mean of the visible values: which keys are seen."""
    L, d = 12, 4
    q, v = orc.randn((L, d), 50), orc.randn((L, d), 51).astype(np.float64)
    k = np.tile(orc.randn((1, d), 52), (L, 1))

    def mean(rows, **kw):
        o, _ = orc.attention_packed(q[:len(rows)], k, v, np.zeros((len(rows), d)), [(0, len(rows), 0, L)], 1, 1, 1.0, **kw)
        for i, js in enumerate(rows):
            want = v[list(js)].astype(np.float32).astype(np.float64).mean(0) if len(js) else np.zeros(d)
            assert np.allclose(o[i], want, rtol=0, atol=1e-12), (i, kw)

    mean([range(L)] * 3)
    mean([range(10), range(11), range(12)], causal=True)  # three queries stand at the last three keys
    mean([[7, 8, 9], [8, 9, 10], [9, 10, 11]], causal=True, window=3)
    mean([[7, 8, 9, 10, 11], [8, 9, 10, 11], [9, 10, 11]], window=3)
    mean([[0, 1, 8, 9], [0, 1, 9, 10], [0, 1, 10, 11]], causal=True, window=2, prefix=[2])
    b = np.full((1, 5), -np.inf)
    b[0, 2] = 0.0  # only the key at the query's own place
    mean([[9], [10], [11]], bias=b, radius=2)
    mean([[], [], []], bias=np.full((1, 1), -np.inf), radius=0)


def _pin_cap_and_bias(orc):
    """Two keys with scores a and 0, capped, then biased: weights 1 / (1 + e^-(c tanh(a / c) + b0 - b1))."""
    d, a, c = 8, 3.0, 2.0
    q = np.zeros((1, d), np.float32)
    q[0, 0] = 1.0
    k = np.zeros((2, d), np.float32)
    k[0, 0] = a
    v = np.zeros((2, d), np.float32)
    v[0, 0] = 1.0
    bias = np.array([[0.5, 0.25, 7.0]])  # distances -1, 0, 1: the query stands at key 1
    o, _ = orc.attention_packed(q, k, v, np.zeros((1, d)), [(0, 1, 0, 2)], 1, 1, 1.0, cap=c, bias=bias, radius=1)
    assert abs(o[0, 0] - 1 / (1 + np.exp(-(c * np.tanh(a / c) + 0.5 - 0.25)))) < 1e-12


def test_masks(orc):
    _pin_masks(orc)


def test_cap_and_bias(orc):
    _pin_cap_and_bias(orc)


def test_first_queries_of_a_longer_row_see_nothing(orc):
    q, k, v, _ = _packed(orc, [6], 1, 1, 4, 60)
    o, tol = orc.attention_packed(q, k, v, np.ones_like(q), [(0, 5, 0, 2)], 1, 1, 1.0, causal=True)
    assert np.all(o[:3] == 0) and np.all(tol[:3] == 0) and np.all(o[5] == 1) and np.any(o[3] != 0)


def _lora(orc):
    x, A, B = orc.randn((9, 7), 70), orc.randn((2, 3, 7), 71), orc.randn((2, 5, 3), 72)
    return x, A, B, np.array([0.5, 2.0]), orc.randn((9, 5), 73)


def _pin_lora(orc):
    x, A, B, f, c0 = _lora(orc)
    seg = [(0, 2, 1, 3), (3, 4, 0, 2), (8, 1, -1, 3)]
    for acc in (True, False):
        y, S = orc.lora(x, A, B, f, seg, c0, acc)
        base = c0.astype(np.float64) if acc else np.zeros((9, 5))
        for t in range(9):
            if t < 2:
                want = base[t] + 2.0 * np.einsum("k,jk,nj->n", x[t].astype(np.float64), A[1], B[1])
            elif 3 <= t < 7:
                want = base[t] + 0.5 * np.einsum("k,jk,nj->n", x[t].astype(np.float64), A[0, :2], B[0, :, :2])
            else:
                want = base[t] if t == 8 else c0[t]
            assert np.allclose(y[t], want, rtol=0, atol=1e-12) and np.all((S[t] > 0) == (t < 2 or 3 <= t < 7))


def test_lora(orc):
    _pin_lora(orc)


@pytest.mark.parametrize("plant,pin", [(20, _pin_masks), (21, _pin_masks), (22, _pin_masks), (23, _pin_cap_and_bias),
                                       (30, _pin_lora), (31, _pin_lora)])
def test_planted_mistakes_fail(orc, plant, pin):
    orc._plant_py = plant
    try:
        with pytest.raises(AssertionError):
            pin(orc)
    finally:
        orc._plant_py = 0
