"""GPU tests of attention over packed sequences against its float64 definition
(Oracle.attention_packed), within the bound that the definition's fp32
evaluation has: every mask, ragged, empty, padded and cached layouts, values
that must not be seen, single tokens, odd head sizes and addresses, offsets past
32 bits, captured and concurrent calls, refusals."""
import threading

import numpy as np
import pytest

import sdhip

gpu = pytest.mark.gpu

UNTOUCHED = 7.0


def bf16_value(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Case:
    """Queries, keys and spans of lq[i] queries against lk[i] keys; gap rows of no sequence between them."""

    def __init__(self, orc, lq, lk, heads, kv, d, seed=1, gap=0, qstd=1.5):
        self.lq, self.lk, self.heads, self.kv, self.d = lq, lk, heads, kv, d
        q0 = np.cumsum([0] + [n + gap for n in lq])
        k0 = np.cumsum([0] + [n + gap for n in lk])
        self.Tq, self.Tk = int(q0[-1]), int(k0[-1])
        self.spans = np.array(list(zip(q0[:-1], lq, k0[:-1], lk)), np.int32).reshape(-1, 4)
        self.q = orc.randn((self.Tq, heads * d), seed, 0.0, qstd)
        self.k, self.v = orc.randn((self.Tk, kv * d), seed + 1), orc.randn((self.Tk, kv * d), seed + 2)
        self.scale = float(np.float32(1) / np.sqrt(np.float32(d)))

    def run(self, be, spans=None, out_bf16=False, k=None, v=None, **kw):
        """The library's result, rows of no sequence holding UNTOUCHED."""
        spans = self.spans if spans is None else spans
        full = np.full(self.q.shape, UNTOUCHED, np.float32)
        out = be.array((full.view(np.uint32) >> 16).astype(np.uint16) if out_bf16 else full)
        kw = {n: be.array(a, a.dtype) if isinstance(a, np.ndarray) else a for n, a in kw.items()}
        be.attention_packed(be.array(self.q), be.array(self.k if k is None else k), be.array(self.v if v is None else v),
                            out, self.Tq, self.Tk, self.heads, self.kv, self.d, be.rows_list(spans), len(spans), self.scale,
                            out_bf16=out_bf16, **kw)
        got = out.download()
        return bf16_value(got) if out_bf16 else got

    def check(self, be, orc, spans=None, out_bf16=False, k=None, v=None, what="", **kw):
        spans = self.spans if spans is None else spans
        got = self.run(be, spans, out_bf16, k, v, **kw)
        want, tol = orc.attention_packed(self.q, self.k if k is None else k, self.v if v is None else v,
                                         np.full(self.q.shape, UNTOUCHED), spans, self.heads, self.kv, self.scale, **kw)
        if out_bf16:
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol) * (tol > 0)
        assert np.all(np.isfinite(got)), what
        over = np.abs(got - want) - tol
        assert np.max(over, initial=0) <= 0, f"{what}: {np.max(over):.3e} beyond the bound at {np.argwhere(over == over.max())[0]}"
        return got


MASKS = {
    "all": {},
    "causal": {"causal": True},
    "window": {"window": 5},
    "causal_window": {"causal": True, "window": 9},
    "prefix": {"causal": True, "prefix": 3},
    "prefix_window": {"causal": True, "window": 4, "prefix": 70},
    "cap": {"causal": True, "cap": 2.0},
    "bias": {"radius": 6},
    "everything": {"causal": True, "window": 40, "prefix": 2, "cap": 30.0, "radius": 100},
}


def masks(orc, name, seqs, heads, seed=90):
    kw = dict(MASKS[name])
    if "prefix" in kw:
        kw["prefix"] = np.array([(kw["prefix"] + i) % (kw["prefix"] + 3) for i in range(seqs)], np.int32)
    if "radius" in kw:
        kw["bias"] = orc.randn((heads, 2 * kw["radius"] + 1), seed)
    return kw


LAYOUTS = {
    "ragged": ([5, 1, 77, 130], [5, 1, 77, 130], 0),
    "empty": ([3, 0, 4, 2, 0], [0, 5, 70, 1, 0], 0),
    "more_queries": ([70, 9, 1], [66, 2, 1], 3),
    "cross": ([40, 1, 33], [129, 64, 200], 5),
}


@gpu
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_masks(be, orc, layout, mask):
    lq, lk, gap = LAYOUTS[layout]
    c = Case(orc, lq, lk, 4, 2, 64, gap=gap)
    c.check(be, orc, what=f"{layout} {mask}", **masks(orc, mask, len(lq), 4))


@gpu
@pytest.mark.parametrize("heads,kv,d", [(2, 2, 40), (2, 1, 80), (4, 1, 128), (3, 3, 33), (2, 2, 7), (2, 1, 160), (1, 1, 260),
                                        (7, 1, 64), (34, 1, 16), (66, 2, 8)])
@pytest.mark.parametrize("mask", ["all", "everything"])
def test_heads(be, orc, heads, kv, d, mask):
    c = Case(orc, [19, 70], [19, 131], heads, kv, d, seed=200 + d)
    c.check(be, orc, what=f"{heads}/{kv} x {d} {mask}", **masks(orc, mask, 2, heads))


@gpu
@pytest.mark.parametrize("heads,kv,d", [(4, 1, 128), (8, 8, 64), (8, 2, 96), (32, 2, 64), (5, 5, 17), (2, 1, 200)])
@pytest.mark.parametrize("mask", ["all", "causal_window", "everything"])
def test_single_tokens(be, orc, heads, kv, d, mask):
    """One query against 0, 1, a few and many keys, in slots."""
    lk = [0, 1, 63, 64, 65, 300, 1031]
    c = Case(orc, [1] * len(lk), lk, heads, kv, d, seed=300 + d, gap=2)
    c.check(be, orc, what=f"{heads}/{kv} x {d} {mask}", **masks(orc, mask, len(lk), heads))
    one = Case(orc, [1], [5003], heads, kv, d, seed=310 + d)
    one.check(be, orc, what=f"one sequence {heads}/{kv} x {d} {mask}", **masks(orc, mask, 1, heads))
    few = Case(orc, [3, 2, 0, 1], [700, 2, 9, 40], heads, kv, d, seed=320 + d)
    few.check(be, orc, what=f"few {heads}/{kv} x {d} {mask}", **masks(orc, mask, 4, heads))


@gpu
def test_many_queries(be, orc):
    """Enough rows for several workgroups a sequence, checked at rows of each."""
    c = Case(orc, [700, 1, 300], [700, 1, 900], 6, 3, 128, seed=400)
    kw = {"causal": True, "window": 333, "cap": 20.0}
    got = c.run(be, **kw)
    for s, (q0, lq, k0, lk) in enumerate(c.spans):
        for i in sorted({0, 1, 31, 85, 86, 255, 256, lq // 2, lq - 1} & set(range(lq))):
            want, tol = orc.attention_packed(c.q[q0 + i:q0 + i + 1], c.k, c.v, np.zeros((1, 768)),
                                             [(0, 1, k0, i + 1 + lk - lq)], 6, 3, c.scale, causal=True, window=333, cap=20.0)
            assert np.all(np.abs(got[q0 + i] - want[0]) <= tol[0]), (s, i)
    full = c.run(be)
    for q0, lq, k0, lk in c.spans:
        for i in sorted({0, lq // 3, lq - 1}):
            want, tol = orc.attention_packed(c.q[q0 + i:q0 + i + 1], c.k, c.v, np.zeros((1, 768)), [(0, 1, k0, lk)], 6, 3, c.scale)
            assert np.all(np.abs(full[q0 + i] - want[0]) <= tol[0]), i


@gpu
@pytest.mark.parametrize("mask", ["all", "everything"])
@pytest.mark.parametrize("lq", [[40, 1, 90], [1, 1, 1]])
def test_bf16_result(be, orc, mask, lq):
    c = Case(orc, lq, [40, 30, 90], 4, 2, 64, seed=500, gap=1)
    c.check(be, orc, out_bf16=True, what=mask, **masks(orc, mask, 3, 4))


@gpu
@pytest.mark.parametrize("lq", [[50, 70], [1, 1]])
@pytest.mark.parametrize("low", [-np.inf, np.finfo(np.float32).min])
@pytest.mark.parametrize("d", [64, 160])
def test_bias_that_hides(be, orc, lq, low, d):
    """Biases of -inf hide keys, all of them give zeros; the type's lowest value on every key weighs them alike."""
    c = Case(orc, lq, [50, 130], 4, 2, d, seed=600)
    bias = orc.randn((4, 31), 601)
    bias[:, 20:] = low
    bias[1, :16] = low  # sees nothing else in front
    bias[2, :] = low
    c.check(be, orc, what=f"{low}", bias=bias, radius=15)
    c.check(be, orc, what=f"causal {low}", bias=bias, radius=15, causal=True)


@gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, 1e30, -3e38])
@pytest.mark.parametrize("lq", [[100, 150], [1, 1], [3, 2]])
@pytest.mark.parametrize("d", [64, 128, 160])
def test_unseen_values(be, orc, bad, lq, d):
    """Keys and values that no query of a row may see change none of its bits' correctness: rows between the
    sequences, keys behind the diagonal, outside the window, in front of it."""
    c = Case(orc, lq, [100, 150], 2, 1, d, seed=700, gap=30)
    k, v = c.k.copy(), c.v.copy()
    inside = np.zeros(c.Tk, bool)
    for _, _, k0, lk in c.spans:
        inside[k0:k0 + lk] = True
    k[~inside] = bad
    v[~inside] = bad
    c.check(be, orc, k=k, v=v, what="gaps")
    c.check(be, orc, k=k, v=v, what="gaps causal", causal=True)
    # the window ends before key 20 of the rows from 60 on; the rows up to 40 end before key 41
    for t in (0, 1):
        k0 = c.spans[t, 2]
        v[k0 + 20] = bad
        k[k0 + 41] = bad
        v[k0 + 47, 3] = bad
    for kw in ({"causal": True, "window": 30}, {"window": 12}):
        got = c.run(be, k=k, v=v, **kw)
        want, tol = orc.attention_packed(c.q, c.k, c.v, np.full(c.q.shape, UNTOUCHED), c.spans, 2, 1, c.scale, **kw)
        clean = 0
        for q0, n, k0, lk in c.spans:
            for i in range(n):
                p = i + lk - n
                lo, hi = p - kw["window"] + 1, p if kw.get("causal") else p + kw["window"] - 1
                if any(lo <= j <= hi for j in (20, 41, 47)):
                    continue
                clean += 1
                assert np.all(np.abs(got[q0 + i] - want[q0 + i]) <= tol[q0 + i]), (kw, i)
        assert clean >= sum(lq) // 5


@gpu
@pytest.mark.parametrize("lq", [[66], [1]])
def test_seen_infinities_stay_in_their_rows(be, orc, lq):
    """A NaN key makes every row that sees it NaN; an infinite value shows in its column; other rows keep their results."""
    c = Case(orc, lq + [70], [66, 70], 2, 2, 64, seed=800)
    k, v = c.k.copy(), c.v.copy()
    k[10, 5] = np.nan
    v[c.spans[1, 2] + 30, 64 + 2] = np.inf
    got = c.run(be, k=k, v=v, causal=True)
    want, tol = orc.attention_packed(c.q, c.k, c.v, np.zeros(c.q.shape), c.spans, 2, 2, c.scale, causal=True)
    for i in range(lq[0]):
        if i + 66 - lq[0] >= 10:
            assert np.all(np.isnan(got[i, :64]))
        else:
            assert np.all(np.abs(got[i, :64] - want[i, :64]) <= tol[i, :64])
        assert np.all(np.abs(got[i, 64:] - want[i, 64:]) <= tol[i, 64:])
    for i in range(70):
        row = lq[0] + i
        ok = np.abs(got[row] - want[row]) <= tol[row]
        if i >= 30:
            assert got[row, 66] == np.inf
            ok[66] = True
        assert np.all(ok), i


@gpu
@pytest.mark.parametrize("lq", [[90], [1]])
def test_wide_scales(be, orc, lq):
    """Keys and values of very unlike size in one sequence."""
    c = Case(orc, lq, [90], 2, 2, 64, seed=850)
    c.k[::7] *= 100.0
    c.v *= np.exp2(np.arange(90) % 24 - 12).astype(np.float32)[:, None]
    c.check(be, orc, what="unlike rows")
    c.v[:] = c.v * np.float32(2.0 ** 60)
    c.check(be, orc, what="large values", causal=True)
    c.v[:] = c.v * np.float32(2.0 ** -120)
    c.check(be, orc, what="small values", causal=True)


@gpu
@pytest.mark.parametrize("d", [64, 40])
@pytest.mark.parametrize("lq", [[60, 33], [1, 1]])
def test_addresses(be, orc, d, lq):
    """Operands at addresses that are multiples of 4 only."""
    c = Case(orc, lq, [60, 33], 2, 2, d, seed=900)
    want, tol = orc.attention_packed(c.q, c.k, c.v, np.zeros(c.q.shape), c.spans, 2, 2, c.scale, causal=True)
    spans = be.rows_list(c.spans)
    for which in range(4):
        arrays, ptr = [], []
        for i, a in enumerate((c.q, c.k, c.v, np.zeros(c.q.shape, np.float32))):
            off = 1 if i == which else 0
            arrays.append(be.array(np.concatenate((np.full(off, 5, np.float32), a.ravel()))))
            ptr.append(arrays[-1].ptr + 4 * off)
        be.attention_packed(*ptr, c.Tq, c.Tk, 2, 2, d, spans, 2, c.scale, causal=True)
        got = arrays[3].download()[1 if which == 3 else 0:].reshape(c.q.shape)
        assert np.all(np.abs(got - want) <= tol), which


@gpu
def test_spans_are_cut_to_the_tensors(be, orc):
    """Entries that leave the tensors are cut; the rest of the batch is as it was."""
    c = Case(orc, [10, 20], [10, 20], 2, 2, 64, seed=1000)
    big = 2 ** 31 - 1
    spans = np.array([(0, 10, 0, 10), (25, big, 15, big), (big, 5, 0, 5), (-5, -3, -big, 7), (12, 3, big, big)], np.int32)
    got = c.run(be, spans=spans)
    want, tol = orc.attention_packed(c.q, c.k, c.v, np.full(c.q.shape, UNTOUCHED), spans, 2, 2, c.scale)
    assert np.all(np.abs(got - want) <= tol)
    pre = np.array([-4, big, 3, 3, 3], np.int32)
    got = c.run(be, spans=spans, causal=True, prefix=pre)
    want, tol = orc.attention_packed(c.q, c.k, c.v, np.full(c.q.shape, UNTOUCHED), spans, 2, 2, c.scale, causal=True, prefix=pre)
    assert np.all(np.abs(got - want) <= tol)


@gpu
@pytest.mark.parametrize("lq", [1, 40])
def test_many_sequences(be, orc, lq):
    """More sequences than a wave has lanes; keys shared by all of them."""
    n = 150
    c = Case(orc, [lq] * n, [3] * n, 2, 1, 64, seed=1100)
    c.spans[::2, 2] = 0
    c.spans[::2, 3] = 37
    c.check(be, orc, causal=True)


@gpu
@pytest.mark.parametrize("lq", [1, 50])
def test_offsets_past_32_bits(be, orc, lq):
    """The last keys of a cache of over 2^32 values."""
    heads, kv, d, L = 2, 1, 128, 90
    Tk = (1 << 25) + 500
    k, v = be.empty((Tk, kv * d)), be.empty((Tk, kv * d))
    c = Case(orc, [lq], [L], heads, kv, d, seed=1200)
    first = Tk - L - 3
    be.upload(k.ptr + first * d * 4, c.k)
    be.upload(v.ptr + first * d * 4, c.v)
    out = be.empty(c.q.shape)
    be.attention_packed(be.array(c.q), k, v, out, lq, Tk, heads, kv, d, be.rows_list(np.array([[0, lq, first, L]], np.int32)), 1,
                        c.scale, causal=True)
    want, tol = orc.attention_packed(c.q, c.k, c.v, np.zeros(c.q.shape), c.spans, heads, kv, c.scale, causal=True)
    assert np.all(np.abs(out.download() - want) <= tol)


@gpu
@pytest.mark.parametrize("lq,lk", [([30, 60], [30, 60]), ([1, 1], [500, 2000]), ([3, 4], [3, 4])])
def test_captured(be, orc, lq, lk):
    """A captured call replayed with other spans and values, the direct call between the replays."""
    c = Case(orc, lq, lk, 4, 2, 64, seed=1300)
    q, k, v, out, spans = be.array(c.q), be.array(c.k), be.array(c.v), be.empty(c.q.shape), be.rows_list(c.spans)

    def call():
        be.attention_packed(q, k, v, out, c.Tq, c.Tk, 4, 2, 64, spans, 2, c.scale, causal=True)

    call()
    be.capture_begin()
    call()
    g = be.capture_end()
    try:
        for rep in range(4):
            sp = c.spans.copy()
            sp[1, 3] -= rep % max(1, lk[1] // 2)
            sp[0, 3] = max(1, sp[0, 3] - 3 * rep)
            c.q[:] = orc.randn(c.q.shape, 1310 + rep)
            q.upload(c.q)
            spans.upload(sp)
            be.call("sdh_zero", out.ptr, out.nbytes)
            be.graph_launch(g)
            got = out.download()
            want, tol = orc.attention_packed(c.q, c.k, c.v, np.zeros(c.q.shape), sp, 4, 2, c.scale, causal=True)
            assert np.all(np.abs(got - want) <= tol), rep
            call()
            assert np.array_equal(out.download(), got), rep
    finally:
        be.graph_destroy(g)


@gpu
def test_two_threads(be, orc):
    """Calls of two threads keep to their own results, bit for bit."""
    cases = [Case(orc, [40, 200], [40, 200], 4, 2, 64, seed=1400), Case(orc, [1] * 5, [900] * 5, 8, 2, 128, seed=1410)]
    alone = [c.run(be, causal=True) for c in cases]
    bad = []

    def work(c, want):
        for _ in range(10):
            if not np.array_equal(c.run(be, causal=True), want):
                bad.append(c.lq)

    ts = [threading.Thread(target=work, args=a) for a in zip(cases, alone)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


@gpu
def test_equal_to_attention(be, orc):
    """Two sequences of one length are sdh_attention's batch."""
    N, S, heads, d = 2, 150, 4, 64
    c = Case(orc, [S] * N, [S] * N, heads, heads, d, seed=1500)
    for causal in (False, True):
        out = be.empty((N * S, heads * d))
        be.attention(be.array(c.q), be.array(c.k), be.array(c.v), out, N, S, S, heads, heads, d, causal)
        _, tol = orc.attention_packed(c.q, c.k, c.v, np.zeros(c.q.shape), c.spans, heads, heads, c.scale, causal)
        assert np.all(np.abs(c.run(be, causal=causal) - out.download()) <= 2 * tol)


@gpu
@pytest.mark.parametrize("radius", [0, 1, 33, 95, 200, 3000])
@pytest.mark.parametrize("heads,kv,d", [(4, 4, 64), (6, 2, 64), (3, 1, 128)])
def test_bias_radii(be, orc, radius, heads, kv, d):
    """Tiles inside the radius, across it and behind it; 3000 is more than the LDS takes."""
    c = Case(orc, [130, 400, 7], [130, 400, 420], heads, kv, d, seed=1700 + radius)
    bias = orc.randn((heads, 2 * radius + 1), 1701, 0.0, 2.0)
    for causal in (False, True):
        c.check(be, orc, what=f"radius {radius} causal {causal}", bias=bias, radius=radius, causal=causal)


@gpu
@pytest.mark.parametrize("cap", [1e-40, 1e-3, 1.0, 8.0, 1e4])
@pytest.mark.parametrize("lq", [1, 150])
def test_caps(be, orc, cap, lq):
    c = Case(orc, [lq, lq], [150, 300], 4, 2, 64, seed=1800, qstd=3.0)
    c.check(be, orc, what=f"cap {cap}", cap=float(np.float32(cap)))
    c.check(be, orc, what=f"cap {cap} bias", cap=float(np.float32(cap)), bias=orc.randn((4, 41), 1801), radius=20)


@gpu
@pytest.mark.parametrize("mask", ["causal", "everything", "prefix_window"])
@pytest.mark.parametrize("heads,kv,d", [(8, 1, 128), (8, 2, 64), (3, 3, 40)])
@pytest.mark.parametrize("lq", [[2, 2, 2], [4, 1, 7], [1, 16, 20]])
def test_a_few_queries_of_long_rows(be, orc, lq, heads, kv, d, mask):
    """Up to sixteen rows a sequence and key/value head, some sequences with more, one with more queries than keys."""
    c = Case(orc, lq, [500, 37, 13], heads, kv, d, seed=1750)
    c.check(be, orc, what=f"{lq} {mask}", **masks(orc, mask, 3, heads))


@gpu
def test_what_the_limits_allow(be, orc):
    """A radius beyond every distance is the whole table's; the list's limit is itself allowed."""
    c = Case(orc, [3], [5], 2, 1, 8, seed=1900)
    c.check(be, orc, bias=orc.randn((2, 2001), 1901), radius=1000)
    spans = np.zeros((65536, 4), np.int32)
    spans[-1] = c.spans[0]
    c.check(be, orc, spans=spans)


def _args(**kw):
    a = dict(q=4096, k=4096, v=4096, out=4096, out_bf16=0, Tq=4, Tk=4, heads=2, kv=2, d=8, spans=4096, seqs=1, scale=1.0,
             causal=0, window=0, prefix=None, cap=0.0, bias=None, radius=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw", [{"Tq": -1}, {"Tk": -1}, {"seqs": -1}, {"window": -1}, {"radius": -1}, {"heads": 0}, {"d": 0},
                                {"d": 1025}, {"heads": 3, "kv": 2}, {"heads": 70000, "kv": 70000}, {"Tk": 1 << 30},
                                {"Tq": 1 << 40}, {"seqs": 1 << 30}, {"radius": 1 << 30}, {"scale": float("nan")},
                                {"cap": -1.0}, {"cap": float("inf")}, {"seqs": 65537},
                                {"heads": 4, "kv": 1, "bias": 4096, "radius": 1 << 28}], ids=str)
def test_refusals_of_sizes(kw):
    """Sizes and numbers are refused before anything else is looked at, with or without a device."""
    lib = sdhip.load_library()
    assert lib.sdh_attention_packed(*_args(**kw)) == sdhip.SDH_ERR_INVALID
    assert b"sdh_attention_packed" in lib.sdh_last_error()


@gpu
def test_refusals_of_pointers(be, orc):
    c = Case(orc, [4], [4], 2, 2, 8, seed=1600)
    q, k, v, out, spans = be.array(c.q), be.array(c.k), be.array(c.v), be.empty(c.q.shape), be.rows_list(c.spans)
    more = be.empty((64,))

    def refused(**kw):
        a = dict(q=q, k=k, v=v, out=out, Tq=4, Tk=4, heads=2, kv_heads=2, d=8, spans=spans, seqs=1, scale=1.0)
        a.update(kw)
        with pytest.raises(sdhip.SdhError) as e:
            be.attention_packed(**a)
        assert e.value.status == sdhip.SDH_ERR_INVALID, kw

    for n in ("q", "k", "v", "out", "spans"):
        refused(**{n: None})
        refused(**{n: 4096})
    refused(Tq=5)
    refused(Tk=5)
    refused(seqs=2)
    refused(out=q)
    refused(out=k.ptr)
    refused(out=v.ptr + 4, Tq=3)
    refused(spans=more.ptr + 4)
    refused(prefix=4096)
    refused(bias=more, radius=16)
    refused(bias=out, radius=3)
    refused(prefix=out)
    be.attention_packed(q, None, None, out, 4, 0, 2, 2, 8, spans, 1, 1.0)  # no keys: zeros
    assert np.all(out.download() == 0)
    out.upload(np.full(out.shape, UNTOUCHED, np.float32))
    be.attention_packed(q, k, v, out, 4, 4, 2, 2, 8, None, 0, 1.0)  # no sequences: nothing
    be.attention_packed(None, None, None, None, 0, 0, 2, 2, 8, None, 0, 1.0)
    assert np.all(out.download() == UNTOUCHED)
