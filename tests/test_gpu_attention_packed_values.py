"""GPU tests of attention over packed sequences at unlike, infinite and undefined values
against its float64 definition (Oracle.attention_packed): keys that are hidden or have no
weight whatever they hold, channels and values of very unlike size, infinities that are
seen, results near fp32's least, and keys cut into several parts."""
import numpy as np
import pytest

from test_gpu_attention_packed import MASKS, UNTOUCHED, Case, masks

gpu = pytest.mark.gpu

# Forty rows go in tiles (up to 128 dims), one and three in the few rows' kernel, 160 dims and more by rows.
SHAPES = [([40], 64), ([40], 128), ([1], 64), ([3], 128), ([1], 40), ([40], 96), ([2], 160)]


def held(c, be, orc, what="", out_bf16=False, **kw):
    """The library's result within the definition's bound; NaN and infinities where the definition has them."""
    got = c.run(be, out_bf16=out_bf16, **kw)
    want, tol = orc.attention_packed(c.q, c.k, c.v, np.full(c.q.shape, UNTOUCHED), c.spans, c.heads, c.kv, c.scale, **kw)
    if out_bf16:
        with np.errstate(invalid="ignore"):
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol) * (tol > 0)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN at {np.argwhere(np.isnan(got) != np.isnan(want))[0]}"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities"
    over = np.abs(got[fin].astype(np.float64) - want[fin]) - tol[fin]
    assert np.max(over, initial=0) <= 0, (f"{what}: {np.max(over):.3e} beyond the bound at {np.argwhere(fin)[np.argmax(over)]}, "
                                          f"bound {tol[fin][np.argmax(over)]:.3e}")
    return got


# ------------------------------------------------- values of keys without weight
@gpu
@pytest.mark.parametrize("big", [1e6, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("lq,d", SHAPES)
def test_large_values_that_a_bias_hides(be, orc, lq, d, big):
    """The last 40 of 150 keys' rows do not see the first 50 keys, some of whose values are large."""
    c = Case(orc, lq, [150], 4, 2, d, seed=2000)
    c.v[[3, 20, 33, 44]] *= np.float32(big)
    bias = orc.randn((4, 301), 2001)
    bias[:, :91] = -np.inf
    held(c, be, orc, f"{big}", bias=bias, radius=150)
    held(c, be, orc, f"{big} causal", bias=bias, radius=150, causal=True)
    c.k[[3, 20, 33, 44]] *= np.float32(big)
    held(c, be, orc, f"{big} with their keys", bias=bias, radius=150)


@gpu
@pytest.mark.parametrize("depth", [20.0, 30.0, 60.0])
@pytest.mark.parametrize("big", [1e6, 1e10, 1e30])
@pytest.mark.parametrize("lq,d", SHAPES)
def test_large_values_of_little_weight(be, orc, lq, d, big, depth):
    """A key whose score lies 20 to 60 below the others', with a large value, alone in its tile or among others."""
    for place in ([20], [100], [20, 21, 100]):
        c = Case(orc, lq, [150], 2, 1, d, seed=2100)
        c.q[:, ::d] = 8.0
        c.k[place, 0] = -depth / (8.0 * c.scale)
        c.v[place] *= np.float32(big)
        held(c, be, orc, f"{place}")
        held(c, be, orc, f"{place} cap", cap=100.0)
        held(c, be, orc, f"{place} bias", bias=orc.randn((2, 61), 2101), radius=30)


@gpu
@pytest.mark.parametrize("lq,d", SHAPES)
def test_the_heaviest_key_has_no_value(be, orc, lq, d):
    """What is left of the others is theirs to the same number of bits."""
    for depth in (5.0, 20.0, 50.0):
        for value in (0.0, 1e-30):
            c = Case(orc, lq, [150], 2, 1, d, seed=2200)
            c.q[:, ::d] = 8.0
            c.k[70, 0] = depth / (8.0 * c.scale)
            c.v[70] *= np.float32(value)
            held(c, be, orc, f"{depth} {value}")


@gpu
@pytest.mark.parametrize("lq,d", SHAPES)
def test_values_that_grow_as_scores_fall(be, orc, lq, d):
    """All keys give alike shares: values from 1 to 2^90 against scores that fall as fast, in either order of keys."""
    for step in (1, -1):
        c = Case(orc, lq, [150], 2, 1, d, seed=2300)
        n = np.arange(150)[::step] * (60.0 / 150)
        c.q[:, ::d] = 8.0
        c.k[:, 0] = -n / (8.0 * c.scale)
        c.v *= np.exp(n).astype(np.float32)[:, None]
        held(c, be, orc, f"{step}")
        held(c, be, orc, f"{step} causal", causal=True)


@gpu
@pytest.mark.parametrize("power", [-60, -100, -110, -116, 60, 100])
@pytest.mark.parametrize("lq,d", SHAPES)
def test_powers_of_two(be, orc, lq, d, power):
    """Values near fp32's least and largest."""
    c = Case(orc, lq, [150], 2, 1, d, seed=2400)
    c.v = (c.v * np.float64(2.0 ** power)).astype(np.float32)
    held(c, be, orc, f"2^{power}")
    held(c, be, orc, f"2^{power} causal", causal=True)


# ----------------------------------------------------------- keys that are not finite
@gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("lq,d", SHAPES)
def test_hidden_by_a_bias_whatever_they_hold(be, orc, lq, d, bad):
    c = Case(orc, lq, [150], 4, 2, d, seed=2500)
    bias = orc.randn((4, 301), 2501)
    bias[:, :91] = -np.inf
    bias[1] = -np.inf  # a head that sees nothing at all
    c.v[[3, 20, 33, 44]] = bad
    held(c, be, orc, f"{bad} values", bias=bias, radius=150)
    c.k[[3, 21, 33, 45]] = bad
    held(c, be, orc, f"{bad}", bias=bias, radius=150)
    held(c, be, orc, f"{bad} causal cap", bias=bias, radius=150, causal=True, cap=30.0)
    one = np.full((4, 1), -np.inf, np.float32)
    assert np.all(held(c, be, orc, "nothing", bias=one, radius=0) == 0)


@gpu
@pytest.mark.parametrize("lq,d", SHAPES)
def test_infinite_keys(be, orc, lq, d):
    """Scores of -inf have no weight, scores of +inf and 0 * inf make their rows NaN, a cap makes both finite."""
    for sign in (1.0, -1.0):
        for where in (0, 1, d - 1):
            c = Case(orc, lq, [150], 2, 2, d, seed=2600)
            c.q[:, where::d] = np.abs(c.q[:, where::d]) + 0.25
            c.k[40, where], c.k[100, d + where] = sign * np.inf, -np.inf
            held(c, be, orc, f"{sign} {where}")
            held(c, be, orc, f"{sign} {where} causal", causal=True)
            held(c, be, orc, f"{sign} {where} cap", cap=5.0)
            held(c, be, orc, f"{sign} {where} bias", bias=orc.randn((2, 21), 2601), radius=10)
    c.q[0, :d] = 0.0
    held(c, be, orc, "0 * inf")
    c.q[0, :d] = np.nan
    held(c, be, orc, "NaN query")
    c.q[0, :d] = 1.0
    c.q[0, 3] = np.inf
    held(c, be, orc, "infinite query")
    held(c, be, orc, "infinite query cap", cap=5.0)


@gpu
@pytest.mark.parametrize("lq,d", SHAPES)
def test_infinite_keys_with_infinite_values(be, orc, lq, d):
    """A score of -inf leaves its value out; under a cap, or with a score that is finite, it shows."""
    c = Case(orc, lq, [150], 2, 2, d, seed=2650)
    c.q[:, 3::d] = np.abs(c.q[:, 3::d]) + 0.25
    c.k[40, 3], c.k[100, d + 3] = -np.inf, -np.inf
    c.v[40] = np.inf
    c.v[100, 1] = np.nan
    for kw in ({}, {"causal": True}, {"cap": 5.0}, {"bias": orc.randn((2, 21), 2651), "radius": 10}):
        held(c, be, orc, str(list(kw)), **kw)


@gpu
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("lq,d", SHAPES)
def test_seen_infinities_of_hardly_any_weight(be, orc, lq, d, value):
    """A key 300 below the others, in front of them, behind them or between them."""
    for place in (0, 75, 149):
        c = Case(orc, lq, [150], 2, 1, d, seed=2700)
        c.q[:, ::d] = 8.0
        c.k[place, 0] = -300.0 / (8.0 * c.scale)
        c.v[place, 2] = value
        c.v[place, d - 1] = value
        held(c, be, orc, f"{place}")
        held(c, be, orc, f"{place} causal", causal=True)


# ------------------------------------------------------------------ unlike channels
@gpu
@pytest.mark.parametrize("power", [12, 24, 40])
@pytest.mark.parametrize("lq,d", SHAPES)
def test_unlike_channels(be, orc, lq, d, power):
    """A channel of the queries, or of the keys, that is far above the others and meets nothing, or next to nothing."""
    up = np.float32(2.0 ** power)
    for meets in (np.float32(0), 1 / up):
        for which in ("q", "k", "both"):
            c = Case(orc, lq, [150], 2, 1, d, seed=2800)
            if which != "k":
                c.q[:, 5::d] *= up
                c.k[:, 5] *= meets
            if which != "q":
                c.k[:, 7] *= up
                c.q[:, 7::d] *= meets
            held(c, be, orc, f"{which} {meets}")
            held(c, be, orc, f"{which} {meets} cap and bias", cap=4.0, bias=orc.randn((2, 61), 2801), radius=30, causal=True)


@gpu
@pytest.mark.parametrize("lq,d", SHAPES)
def test_keys_far_above_the_others(be, orc, lq, d):
    """One in each tile, with the others' values or with few."""
    for up in (1e4, 1e8):
        c = Case(orc, lq, [150], 2, 1, d, seed=2850)
        c.k[::64] *= np.float32(up)
        held(c, be, orc, f"{up}")
        held(c, be, orc, f"{up} causal", causal=True)
        c.k[::64, : d // 2] *= np.float32(1 / up)
        held(c, be, orc, f"{up} half")


# --------------------------------------------------------------- keys cut into parts
def parts_of_tiles(c, cus=256):
    """How many parts the dispatch cuts the keys into: those that fill the chip, of 512 keys of an average sequence at least."""
    group, waves = c.heads // c.kv, 8 if c.d > 64 else 4
    live = min(len(c.spans), c.Tq)
    assert -(-c.Tq // live) * group > 16, "the few rows' kernel"
    wgs = (c.Tq * group // (32 * waves) + live) * c.kv
    return min(cus * (8 // waves) // wgs, c.Tk // len(c.spans) // 512, 256)


PART_SHAPES = [(4, 1, 128), (8, 2, 64), (2, 2, 40)]


@gpu
@pytest.mark.parametrize("mask", list(MASKS) + ["long_prefix"])
@pytest.mark.parametrize("heads,kv,d", PART_SHAPES)
def test_parts(be, orc, heads, kv, d, mask):
    """Some tens of rows against thousands of keys."""
    c = Case(orc, [24, 33], [3000, 4500], heads, kv, d, seed=2900, gap=1)
    assert parts_of_tiles(c) >= 4
    kw = {"causal": True, "window": 900, "prefix": np.array([1500, 2777], np.int32)} if mask == "long_prefix" else masks(orc, mask, 2, heads)
    for out_bf16 in (False, True):
        held(c, be, orc, f"{mask} bf16 {out_bf16}", out_bf16, **kw)


@gpu
@pytest.mark.parametrize("lq", [[24, 33], [1, 1]])
@pytest.mark.parametrize("heads,kv,d", PART_SHAPES)
def test_parts_of_unlike_values(be, orc, heads, kv, d, lq):
    """What one part holds: large values, hidden or of little weight, infinities of hardly any, keys that are not finite."""
    def case(seed=3000):
        c = Case(orc, lq, [3000, 4500], heads, kv, d, seed=seed)
        c.q[:, ::d] = 8.0
        return c

    def low(c, j, depth):
        c.k[j, 0] = -depth / (8.0 * c.scale)

    for depth, value in ((30.0, 1e10), (60.0, 1e30)):
        c = case()
        low(c, [700, 3000 + 2000], depth)
        c.v[[700, 3000 + 2000]] *= np.float32(value)
        held(c, be, orc, f"{depth} {value}")
    c = case()
    low(c, [700, 3000 + 2000], 300.0)
    c.v[700, 3], c.v[3000 + 2000, 5] = np.inf, np.nan
    held(c, be, orc, "infinity of hardly any weight")
    c = case()
    c.q[:, 3::d] = np.abs(c.q[:, 3::d]) + 0.25
    c.k[700, 3], c.k[3000 + 2000, 3] = -np.inf, -np.inf
    c.v[700] = np.inf
    held(c, be, orc, "scores of -inf")
    c.k[800, 3] = np.nan
    held(c, be, orc, "a NaN key")
    c = case()
    c.v = (c.v * np.float64(2.0 ** -112)).astype(np.float32)
    held(c, be, orc, "least values")
    c = case()
    low(c, np.arange(0, 1500), 100.0)
    c.v[:1500] = 0
    c.v[1500:3000] *= np.float32(2.0 ** -40)
    held(c, be, orc, "parts of no value and no weight")


@gpu
@pytest.mark.parametrize("lq", [[24, 33], [1, 1]])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 1e30])
def test_parts_that_a_bias_hides(be, orc, lq, bad):
    c = Case(orc, lq, [3000, 4500], 4, 1, 128, seed=3100)
    bias = orc.randn((4, 2 * 2500 + 1), 3101)
    bias[:, :1200] = -np.inf  # more than 1300 in front
    c.v[:1600] = bad
    c.k[100:1500] = bad
    c.v[3000:3000 + 3000] = bad
    held(c, be, orc, f"{bad}", bias=bias, radius=2500)
    held(c, be, orc, f"{bad} window", bias=bias, radius=2500, causal=True, window=2000)


# ------------------------------------------------- tiles that wait, among many that do not
@gpu
@pytest.mark.parametrize("kw", [{}, {"causal": True}, {"causal": True, "window": 300, "prefix": 70, "cap": 20.0}], ids=str)
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 128), (2, 2, 64), (2, 1, 72)])
def test_odd_tiles_among_others(be, orc, heads, kv, d, kw):
    """Keys and values of unlike size, rows of zeros, keys that are not finite and infinite values in some tiles of
    sequences of several workgroups, checked at rows of each."""
    lens = [700, 130, 1000]
    c = Case(orc, lens, lens, heads, kv, d, seed=3200, gap=3)
    first = c.spans[:, 2]
    c.k[first[0] + 70] *= np.float32(2.0 ** 14)     # the second tile
    c.v[first[0] + 200] *= np.float32(2.0 ** -20)   # the fourth
    c.v[first[0] + 390:first[0] + 400] = 0.0        # the seventh
    c.v[first[1]] *= np.float32(1e-6)               # a first key that gives next to nothing
    c.q[:, 3::d] = np.abs(c.q[:, 3::d]) + 0.25
    c.k[first[2] + 500, 3] = -np.inf
    c.k[first[2] + 640, d * (kv - 1) + 5] = np.nan  # rows that see it are NaN, in their heads
    c.v[first[2] + 333, 7] = np.inf
    c.q[first[2] + 900] = 0.0                       # a zero query: 0 * inf
    pre = kw.get("prefix")
    kw = dict(kw, prefix=np.array([pre, 0, pre + 30], np.int32)) if pre else kw
    got = c.run(be, **kw)
    for s, n in enumerate(lens):
        for i in sorted({0, 1, 31, 32, 63, 64, 127, 128, 255, 256, 333, 334, 390, 499, 500, 639, 640, 699, 900, n // 2, n - 1} & set(range(n))):
            one = dict(kw, prefix=kw["prefix"][s:s + 1]) if pre else kw
            row = first[s] + i
            # the row alone, with the keys up to its own place or, not causal, all of its sequence's
            keys = i + 1 if kw.get("causal") else n
            if pre and keys < one["prefix"][0]:
                continue  # it sees keys behind its place, which a row alone cannot
            want, tol = orc.attention_packed(c.q[row:row + 1], c.k, c.v, np.zeros((1, heads * d)), [(0, 1, first[s], keys)], heads, kv,
                                             c.scale, **one)
            fin = np.isfinite(want[0])
            assert np.array_equal(np.isnan(got[row]), np.isnan(want[0])), (s, i)
            assert np.array_equal(got[row][np.isinf(want[0])], want[0][np.isinf(want[0])]), (s, i)
            assert np.all(np.abs(got[row][fin] - want[0][fin]) <= tol[0][fin]), (s, i)
    again = c.run(be, **kw)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32))


@gpu
@pytest.mark.parametrize("lq,lk", [([30, 260], [150, 260]), ([1, 1], [500, 2000]), ([24, 33], [3000, 4500])])
def test_captured_with_unlike_values(be, orc, lq, lk):
    """Replayed with values that send other tiles to the second loop, the direct call between the replays."""
    c = Case(orc, lq, lk, 4, 1, 128, seed=3300)
    q, k, v, out, spans = be.array(c.q), be.array(c.k), be.array(c.v), be.empty(c.q.shape), be.rows_list(c.spans)

    def call():
        be.attention_packed(q, k, v, out, c.Tq, c.Tk, 4, 1, 128, spans, 2, c.scale, causal=True)

    call()
    be.capture_begin()
    call()
    g = be.capture_end()
    try:
        for rep in range(4):
            hk, hv = c.k.copy(), c.v.copy()
            hv[rep * 30 + 5] *= np.float32(1e-5)
            hk[rep * 20 + 3] *= np.float32(1e5)
            if rep % 2:
                hv[7, 3], hk[lk[0] + 100, 2] = np.inf, np.nan
            k.upload(hk)
            v.upload(hv)
            be.call("sdh_zero", out.ptr, out.nbytes)
            be.graph_launch(g)
            got = out.download()
            want, tol = orc.attention_packed(c.q, hk, hv, np.zeros(c.q.shape), c.spans, 4, 1, c.scale, causal=True)
            fin = np.isfinite(want)
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), rep
            assert np.all(np.abs(got[fin] - want[fin]) <= tol[fin]), rep
            call()
            assert np.array_equal(out.download().view(np.uint32), got.view(np.uint32)), rep
    finally:
        be.graph_destroy(g)
