"""GPU tests of low-rank adapters of many requests (sdh_lora_nt_*) against their
float64 definition (Oracle.lora) within the rigorous fp32 summation bound: types,
odd sizes, strides, ranks, runs without an adapter, rows of no run, entries past
the matrix, captured and concurrent calls, refusals."""
import threading

import numpy as np
import pytest

import sdhip

gpu = pytest.mark.gpu

UNTOUCHED = 7.0
TYPES = ["f32_bf16", "bf16_bf16", "f32_f32"]


def f32_to_bf16(a):
    from oracle import f32_to_bf16 as f

    return f(a).reshape(np.shape(a))


def bf16_value(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Case:
    def __init__(self, orc, M, N, K, rank, adapters, types="f32_bf16", seed=1, pad=0):
        self.M, self.N, self.K, self.rank, self.adapters, self.types = M, N, K, rank, adapters, types
        self.ldx, self.ldc = K + pad, N + pad
        self.x = orc.randn((M, self.ldx), seed)
        self.A = orc.randn((adapters, rank, K), seed + 1, 0.0, 1 / np.sqrt(K))
        self.B = orc.randn((adapters, N, rank), seed + 2, 0.0, 1 / np.sqrt(rank))
        self.scale = orc.randn((adapters,), seed + 3)
        self.c0 = orc.randn((M, self.ldc), seed + 4)
        if types.startswith("bf16"):
            self.x = bf16_value(f32_to_bf16(self.x))
        if types.endswith("bf16"):
            self.A, self.B = bf16_value(f32_to_bf16(self.A)), bf16_value(f32_to_bf16(self.B))

    def device(self, be):
        up = lambda a, h: be.array(f32_to_bf16(a) if h else a)  # noqa: E731
        x16, w16 = (t == "bf16" for t in self.types.split("_"))
        return up(self.x, x16), up(self.A, w16), up(self.B, w16), be.array(self.scale)

    def call(self, be, X, A, B, scale, runs, n, C, accumulate):
        f = {"f32_bf16": be.lora_nt_bf16, "bf16_bf16": be.lora_nt_bf16_packed, "f32_f32": be.lora_nt_f32}[self.types]
        f(self.M, self.N, self.K, X, self.ldx, A, B, self.rank, self.adapters, scale, runs, n, C, self.ldc, accumulate)

    def check(self, be, orc, runs, accumulate=True, scaled=True, what=""):
        runs = np.array(runs, np.int32).reshape(-1, 4)
        X, A, B, scale = self.device(be)
        C = be.array(self.c0)
        self.call(be, X, A, B, scale if scaled else None, be.rows_list(runs), len(runs), C, accumulate)
        got = C.download()
        self.compare(orc, got, runs, accumulate, scaled, what)
        return got

    def compare(self, orc, got, runs, accumulate=True, scaled=True, what=""):
        with np.errstate(invalid="ignore", over="ignore"):
            want, tol = orc.lora(self.x[:, :self.K], self.A, self.B, self.scale if scaled else None, runs,
                                 self.c0[:, :self.N], accumulate)
        over = np.abs(got[:, :self.N] - want) - tol
        assert np.all(over <= 0), f"{what}: {np.nanmax(over):.3e} beyond the bound at {np.argwhere(~(over <= 0))[0]}"
        assert np.array_equal(got[:, self.N:], self.c0[:, self.N:]), what


def ragged(rows, adapters, rank, seed=3):
    """Runs of the given rows, adapters in turn with -1 among them, ranks from 0 up to the full one."""
    out, first = [], 0
    for i, n in enumerate(rows):
        out.append((first, n, i % (adapters + 1) - 1 if i else 0, (rank, rank, (rank + 1) // 2, 1, 0)[i % 5]))
        first += n
    return out


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("N,K,rank", [(256, 128, 16), (1000, 650, 8), (33, 7, 3), (4096, 320, 64), (300, 1288, 21), (1, 1, 1),
                                      (515, 512, 128), (96, 64, 200)])
def test_sizes(be, orc, types, N, K, rank):
    rows = [1, 5, 0, 64, 1, 33, 130, 2, 17]
    c = Case(orc, sum(rows), N, K, rank, 3, types, seed=100 + K)
    for acc in (True, False):
        c.check(be, orc, ragged(rows, 3, rank), acc, what=f"{types} {N}x{K} rank {rank} acc={acc}")


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [[1], [1] * 9, [2, 1, 1, 3], [300], [4, 4, 4, 4, 4, 4, 4]])
def test_few_rows(be, orc, types, rows):
    for N, K, rank in ((1024, 256, 8), (2560, 3840, 16), (77, 2500, 33)):
        c = Case(orc, sum(rows), N, K, rank, 4, types, seed=200 + K)
        for acc in (True, False):
            c.check(be, orc, ragged(rows, 4, rank), acc, what=f"{types} {rows} {N}x{K} rank {rank} acc={acc}")


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("N,K,rank", [(1024, 64, 24), (515, 600, 40), (640, 640, 64), (130, 33, 5), (5, 640, 65), (260, 648, 64)])
def test_few_rows_of_a_short_k(be, orc, types, N, K, rank):
    """Both sides of the one-launch route: ranks to 64, K to 640; runs of 0 to 70 rows among them."""
    for rows in ([1, 0, 70, 1, 3, 1, 1, 5], [33]):
        c = Case(orc, sum(rows), N, K, rank, 3, types, seed=250 + K)
        for acc in (True, False):
            c.check(be, orc, ragged(rows, 3, rank), acc, what=f"{types} {rows} {N}x{K} rank {rank} acc={acc}")


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rank,r", [(64, 33), (64, 57), (64, 5), (128, 70), (128, 64), (40, 37), (200, 131), (192, 129)])
@pytest.mark.parametrize("K", [256, 1288])
def test_ranks_that_do_not_count(be, orc, types, rank, r, K):
    """NaN in the rows of A and columns of B behind a run's ranks, few and many rows, one launch and several."""
    for rows in ([1, 3], [90, 170]):
        c = Case(orc, sum(rows), 300, K, rank, 2, types, seed=270 + rank)
        runs = np.array([(0, rows[0], 0, r), (rows[0], rows[1], 1, max(1, r - 9))], np.int32)
        for a, n in ((0, r), (1, max(1, r - 9))):
            c.A[a, n:] = np.nan
            c.B[a, :, n:] = np.nan
        for acc in (True, False):
            c.check(be, orc, runs, acc, what=f"{types} {rows} rank {r} of {rank} acc={acc}")


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("pad", [1, 4, 8])
def test_strides(be, orc, types, pad):
    for rows in ([40, 90, 3], [1, 1]):
        c = Case(orc, sum(rows), 256, 320, 16, 2, types, seed=300, pad=pad)
        c.check(be, orc, ragged(rows, 2, 16), what=f"{types} +{pad}")
        c.check(be, orc, ragged(rows, 2, 16), False, what=f"{types} +{pad}")


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("which", range(4))
def test_addresses(be, orc, types, which):
    """Operands at addresses that are multiples of their element only."""
    for rows in ([70, 20], [1, 1, 1]):
        c = Case(orc, sum(rows), 128, 256, 16, 2, types, seed=400)
        runs = np.array(ragged(rows, 2, 16), np.int32)
        held, ptr = [], []
        for i, (a, h) in enumerate(((c.x, types.startswith("bf16")), (c.A, types.endswith("bf16")), (c.B, types.endswith("bf16")),
                                    (c.c0, False))):
            off = 1 if i == which else 0
            flat = np.concatenate((np.zeros(off, np.float32), a.ravel()))
            held.append(be.array(f32_to_bf16(flat) if h else flat))
            ptr.append(held[-1].ptr + off * (2 if h else 4))
        c.call(be, ptr[0], ptr[1], ptr[2], be.array(c.scale), be.rows_list(runs), len(runs), ptr[3], True)
        c.compare(orc, held[3].download()[1 if which == 3 else 0:].reshape(c.c0.shape), runs, what=f"{types} {which}")


@gpu
@pytest.mark.parametrize("types", TYPES)
def test_rows_of_no_run_and_entries_past_the_matrix(be, orc, types):
    big = 2 ** 31 - 1
    c = Case(orc, 60, 130, 96, 8, 3, types, seed=500)
    runs = [(3, 7, 0, 8), (20, 1, 2, big), (50, big, 1, 3), (big, 4, 0, 8), (-7, -2, 1, 8), (30, 5, 3, 8), (36, 2, -big, 8), (40, 3, 1, -5)]
    for acc in (True, False):
        for scaled in (True, False):
            c.check(be, orc, runs, acc, scaled, what=f"acc={acc}")
    got = c.check(be, orc, runs)
    assert np.array_equal(got[11:20], c.c0[11:20]) and np.array_equal(got[30:35], c.c0[30:35])


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [[40, 90], [1, 1]])
def test_unread_values(be, orc, types, rows):
    """Ranks that do not count, adapters of no run and rows of no run may hold anything."""
    c = Case(orc, sum(rows) + 5, 200, 128, 12, 3, types, seed=600)
    runs = [(0, rows[0], 0, 5), (rows[0], rows[1], 1, 12)]
    for bad in (np.nan, np.inf):
        c.A[0, 5:], c.B[0, :, 5:], c.A[2], c.B[2], c.x[-5:], c.scale[2] = bad, bad, bad, bad, bad, bad
        got = c.check(be, orc, runs, what=str(bad))
        assert np.all(np.isfinite(got))
        c.check(be, orc, runs, False, what=str(bad))


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [[40, 90], [1, 2]])
def test_values_that_are_not_finite_stay_in_their_rows(be, orc, types, rows):
    c = Case(orc, sum(rows), 200, 128, 12, 2, types, seed=650)
    runs = np.array([(0, rows[0], 0, 12), (rows[0], rows[1], 1, 12)], np.int32)
    clean = c.check(be, orc, runs)
    c.x[0, 9] = np.nan
    c.x[rows[0], 3] = np.inf
    X, A, B, scale = c.device(be)
    C = be.array(c.c0)
    c.call(be, X, A, B, scale, be.rows_list(runs), 2, C, True)
    got = C.download()
    for t in range(sum(rows)):
        if t in (0, rows[0]):
            assert not np.any(np.isfinite(got[t]))
        else:
            assert np.array_equal(got[t], clean[t]), t


@gpu
@pytest.mark.parametrize("types", TYPES)
def test_wide_scales(be, orc, types):
    """fp32's range is kept: rows and weights of very unlike size."""
    for rows in ([40, 90], [1, 2]):
        c = Case(orc, sum(rows), 200, 128, 12, 2, types, seed=700)
        up = np.exp2(np.arange(sum(rows)) % 40 * 2 - 40).astype(np.float32)[:, None]
        c.x *= up
        c.A *= np.float32(2.0 ** -30)
        c.B *= np.float32(2.0 ** 20)
        c.check(be, orc, ragged(rows, 2, 12), False, what=types)


@gpu
@pytest.mark.parametrize("types", TYPES)
def test_many_runs(be, orc, types):
    rows = [1 + i % 3 for i in range(200)]
    c = Case(orc, sum(rows), 96, 64, 8, 5, types, seed=800)
    c.check(be, orc, ragged(rows, 5, 8))


@gpu
@pytest.mark.parametrize("K", [64, 1280])
def test_as_many_runs_as_are_allowed(be, orc, K):
    c = Case(orc, 40, 128, K, 8, 2, seed=850)
    runs = np.zeros((65536, 4), np.int32)
    runs[[7, 40000, 65535]] = [(0, 20, 0, 8), (20, 15, 1, 5), (35, 5, 1, 8)]
    c.check(be, orc, runs)
    c.check(be, orc, runs, False)


@gpu
@pytest.mark.parametrize("rows", [[200, 100], [1, 1, 1]])
def test_captured(be, orc, rows):
    """Replayed with other runs and rows, the direct call between the replays."""
    c = Case(orc, sum(rows), 512, 256, 16, 3, seed=900)
    X, A, B, scale = c.device(be)
    C, seg = be.array(c.c0), be.rows_list(np.array(ragged(rows, 3, 16), np.int32))
    c.call(be, X, A, B, scale, seg, len(rows), C, True)
    be.capture_begin()
    c.call(be, X, A, B, scale, seg, len(rows), C, True)
    g = be.capture_end()
    try:
        for rep in range(4):
            runs = np.array(ragged(rows, 3, 16), np.int32)
            runs[:, 2] = (runs[:, 2] + 1 + rep) % 4 - 1
            c.x[:] = orc.randn(c.x.shape, 910 + rep)
            X.upload(c.x)
            seg.upload(runs)
            C.upload(c.c0)
            be.graph_launch(g)
            got = C.download()
            c.compare(orc, got, runs, what=f"replay {rep}")
            C.upload(c.c0)
            c.call(be, X, A, B, scale, seg, len(rows), C, True)
            assert np.array_equal(C.download(), got), rep
    finally:
        be.graph_destroy(g)


@gpu
def test_two_threads(be, orc):
    cases = [Case(orc, 300, 512, 256, 16, 3, seed=1000), Case(orc, 6, 2560, 1280, 8, 3, "f32_f32", seed=1010)]
    runs = [ragged([200, 100], 3, 16), ragged([1] * 6, 3, 8)]
    alone = [c.check(be, orc, r) for c, r in zip(cases, runs)]
    bad = []

    def work(c, r, want):
        X, A, B, scale = c.device(be)
        for _ in range(10):
            C = be.array(c.c0)
            c.call(be, X, A, B, scale, be.rows_list(np.array(r, np.int32)), len(r), C, True)
            if not np.array_equal(C.download(), want):
                bad.append(c.M)

    ts = [threading.Thread(target=work, args=a) for a in zip(cases, runs, alone)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


@gpu
def test_beside_a_projection(be, orc):
    """Before the shared projection (which then accumulates) and after it: the same rows."""
    c = Case(orc, 130, 256, 320, 16, 2, "bf16_bf16", seed=1100)
    runs = np.array(ragged([100, 30], 2, 16), np.int32)
    W = f32_to_bf16(orc.randn((c.N, c.K), 1101, 0.0, 1 / np.sqrt(c.K)))
    X, A, B, scale = c.device(be)
    dW, seg = be.array(W), be.rows_list(runs)
    before, after = be.empty((c.M, c.N)), be.empty((c.M, c.N))
    be.gemm_nt_bf16_packed(c.M, c.N, c.K, X, c.K, dW, c.K, after, c.N)
    c.call(be, X, A, B, scale, seg, 2, after, True)
    c.call(be, X, A, B, scale, seg, 2, before, False)
    be.gemm_nt_bf16_packed(c.M, c.N, c.K, X, c.K, dW, c.K, before, c.N, None, True)
    base = c.x.astype(np.float64) @ bf16_value(W).astype(np.float64).T
    want, tol = orc.lora(c.x, c.A, c.B, c.scale, runs, base, True)
    tol = tol + (c.K + 2) * 2.0 ** -24 * (np.abs(c.x).astype(np.float64) @ np.abs(bf16_value(W)).T)
    for y in (before, after):
        assert np.all(np.abs(y.download() - want) <= tol)


def _args(**kw):
    a = dict(M=4, N=8, K=8, X=4096, ldx=8, A=4096, B=4096, rank=2, adapters=1, scale=None, runs=4096, n=1, C=4096, ldc=8, acc=1)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("name", ["sdh_lora_nt_bf16", "sdh_lora_nt_bf16_packed", "sdh_lora_nt_f32"])
@pytest.mark.parametrize("kw", [{"M": -1}, {"N": -1}, {"K": -1}, {"rank": -1}, {"adapters": -1}, {"n": -1}, {"ldx": 7}, {"ldc": 7},
                                {"rank": 1025}, {"M": 1 << 30}, {"N": 1 << 30, "ldc": 1 << 30}, {"n": 1 << 31},
                                {"adapters": 1 << 30}, {"K": 1 << 30, "ldx": 1 << 30}, {"n": 65537}, {"ldx": 1 << 45},
                                {"ldc": 1 << 45}, {"adapters": 1 << 29, "N": 1 << 29, "ldc": 1 << 29}], ids=str)
def test_refusals_of_sizes(name, kw):
    lib = sdhip.load_library()
    assert getattr(lib, name)(*_args(**kw)) == sdhip.SDH_ERR_INVALID
    assert name.encode() in lib.sdh_last_error()


@gpu
def test_refusals_of_pointers(be, orc):
    c = Case(orc, 6, 16, 8, 4, 2, seed=1200)
    X, A, B, scale = c.device(be)
    C, seg = be.array(c.c0), be.rows_list(np.array([(0, 6, 0, 4)], np.int32))

    def refused(**kw):
        a = dict(M=6, N=16, K=8, X=X, ldx=8, A=A, B=B, rank=4, adapters=2, scale=scale, segments=seg, count=1, C=C, ldc=16)
        a.update(kw)
        with pytest.raises(sdhip.SdhError) as e:
            be.lora_nt_bf16(**a)
        assert e.value.status == sdhip.SDH_ERR_INVALID, kw

    for n in ("X", "A", "B", "segments", "C"):
        refused(**{n: None})
        refused(**{n: 4096})
    refused(scale=4096)
    refused(M=7)
    refused(adapters=3)
    refused(rank=5)
    refused(count=2)
    refused(ldc=17)
    refused(C=X)
    refused(C=A)
    refused(C=scale)
    refused(C=seg)
    refused(segments=C.ptr + 4)
    be.lora_nt_bf16(6, 16, 8, X, 8, A, B, 4, 2, scale, None, 0, C, 16)  # no runs
    be.lora_nt_bf16(0, 16, 8, None, 8, A, B, 4, 2, scale, seg, 1, None, 16)  # no rows
    be.lora_nt_bf16(6, 16, 8, X, 8, None, None, 4, 0, None, seg, 1, C, 16)  # no adapters: nothing is added
    assert np.array_equal(C.download(), c.c0)
    be.lora_nt_bf16(6, 16, 0, None, 8, None, None, 4, 2, None, seg, 1, C, 16, accumulate=False)  # empty sums
    assert np.all(C.download() == 0)
