"""GPU tests of low-rank adapters (sdh_lora_nt_*) at infinities, against the float64
definition (Oracle.lora), and at offsets past 32 bits and without ranks for many rows."""
import numpy as np
import pytest

from test_gpu_lora import TYPES, Case, bf16_value, f32_to_bf16, ragged

gpu = pytest.mark.gpu


def held(c, be, orc, runs, accumulate, what):
    """The bound where the definition is finite; its infinities and NaN elsewhere."""
    runs = np.array(runs, np.int32).reshape(-1, 4)
    X, A, B, scale = c.device(be)
    C = be.array(c.c0)
    c.call(be, X, A, B, scale, be.rows_list(runs), len(runs), C, accumulate)
    got = C.download()[:, :c.N]
    with np.errstate(invalid="ignore", over="ignore"):
        want, tol = orc.lora(c.x[:, :c.K], c.A, c.B, c.scale, runs, c.c0[:, :c.N], accumulate)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN at {np.argwhere(np.isnan(got) != np.isnan(want))[0]}"
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), f"{what}: infinities"
    assert np.all(np.abs(got[fin] - want[fin]) <= tol[fin]), what
    return want


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [[90, 170], [1, 2]])
@pytest.mark.parametrize("N,K,rank", [(300, 256, 12), (128, 650, 64), (131, 1288, 130), (260, 320, 1)])
def test_infinities(be, orc, types, rows, N, K, rank):
    """An infinity in X is one in its row's results, of the products' sign; it is NaN where signs meet or a zero does.
    So is one in A."""
    runs = [(0, rows[0], 0, rank), (rows[0], rows[1], 1, max(1, rank - 3))]
    for sign in (1.0, -1.0):
        for acc in (True, False):
            c = Case(orc, sum(rows), N, K, rank, 2, types, seed=1300 + K)
            c.A[:, :, 9] = np.abs(c.A[:, :, 9]) + 0.25  # H of those rows has one sign
            c.B[0] = np.abs(c.B[0]) + 0.25
            c.B[1, :N // 2] = -np.abs(c.B[1, :N // 2]) - 0.25  # and random signs behind: NaN there, beyond rank 1
            if types.endswith("bf16"):
                c.A, c.B = bf16_value(f32_to_bf16(c.A)), bf16_value(f32_to_bf16(c.B))
            c.x[0, 9] = sign * np.inf
            c.x[rows[0], 9] = -sign * np.inf
            want = held(c, be, orc, runs, acc, f"{types} {rows} {N}x{K} rank {rank} {sign} acc={acc}")
            assert np.all(np.isinf(want[0])) and np.all(np.isinf(want[rows[0], :N // 2]))
            c.x[0, 9], c.x[rows[0], 9] = 1.0, np.nan
            c.A[0, 0, 11] = sign * np.inf
            c.x[:, 11] = np.abs(c.x[:, 11]) + 0.25
            if types.startswith("bf16"):
                c.x = bf16_value(f32_to_bf16(c.x))
            held(c, be, orc, runs, acc, f"{types} infinite A acc={acc}")


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [[90, 0, 170, 40], [600, 3]])
def test_no_ranks_for_many_rows(be, orc, types, rows):
    """Rows without an adapter, adapters without ranks, and no adapters at all: left, or zero without accumulate."""
    c = Case(orc, sum(rows), 260, 128, 16, 2, types, seed=1400)
    first = np.cumsum([0] + rows[:-1])
    for acc in (True, False):
        for a, r in ((-1, 16), (0, 0), (2, 16), (1, -3)):
            got = c.check(be, orc, [(f, n, a, r) for f, n in zip(first, rows)], acc, what=f"{a} {r} acc={acc}")
            assert np.array_equal(got, c.c0) if acc else np.all(got == 0)
        c.check(be, orc, [(f, n, i % 2 - 1, 16) for i, (f, n) in enumerate(zip(first, rows))], acc, what=f"mixed acc={acc}")
        for rank, adapters in ((0, 2), (16, 0), (0, 0)):
            C, seg = be.array(c.c0), be.rows_list(np.array([(f, n, 0, 16) for f, n in zip(first, rows)], np.int32))
            f = {"f32_bf16": be.lora_nt_bf16, "bf16_bf16": be.lora_nt_bf16_packed, "f32_f32": be.lora_nt_f32}[types]
            f(c.M, c.N, c.K, None, c.ldx, None, None, rank, adapters, None, seg, len(rows), C, c.ldc, acc)
            got = C.download()
            assert np.array_equal(got, c.c0) if acc else np.all(got == 0)


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("N,K,rank", [(128, 128, 8), (1288, 1280, 64)])
@pytest.mark.parametrize("M", [3, 300])
def test_offsets_past_32_bits(be, orc, types, M, N, K, rank):
    """Rows of X and C, and adapters, whose offsets pass 2^32 values; few rows in one launch and in two, and many."""
    apart = (1 << 32) // (M - 1) // 8 * 8 + 64
    runs = np.array([(0, 1, 1, rank), (1, M - 1, 0, rank)], np.int32)
    c = Case(orc, M, N, K, rank, 2, types, seed=1500)
    X, A, B, scale = c.device(be)
    seg = be.rows_list(runs)
    x16 = types.startswith("bf16")
    w = np.uint16 if types.endswith("bf16") else np.float32
    at = sorted({0, 1, M // 2, M - 1})
    for acc in (True, False):
        C = be.empty(((M - 1) * apart + N,))
        for t in range(M):
            be.upload(C.ptr + t * apart * 4, c.c0[t])
        c.ldc = apart
        c.call(be, X, A, B, scale, seg, 2, C, acc)
        want, tol = orc.lora(c.x, c.A, c.B, c.scale, runs, c.c0, acc)
        for t in at:
            got = np.empty(N, np.float32)
            be.download(got, C.ptr + t * apart * 4)
            assert np.all(np.abs(got - want[t]) <= tol[t]), (t, acc)
        C.free()
    c.ldc = N
    far = be.empty((((M - 1) * apart + K + 1) // (2 if x16 else 1),))
    for t in range(M):
        be.upload(far.ptr + t * apart * (2 if x16 else 4), f32_to_bf16(c.x[t]) if x16 else c.x[t])
    c.ldx = apart
    C = be.array(c.c0)
    c.call(be, far, A, B, scale, seg, 2, C, True)
    want, tol = orc.lora(c.x, c.A, c.B, c.scale, runs, c.c0, True)
    assert np.all(np.abs(C.download() - want) <= tol)
    far.free()
    c.ldx = K
    # adapter n - 1 of n, whose rows of A (or B) start behind 2^32 values
    n = (1 << 32) // (rank * min(K, N)) + 2
    size = np.dtype(w).itemsize
    far = [be.empty((n * rank * s * size // 4 + 1,)) for s in (K, N)]
    for f, host, s in zip(far, (c.A[1], c.B[1]), (K, N)):
        be.upload(f.ptr + (n - 1) * rank * s * size, f32_to_bf16(host) if w == np.uint16 else host)
    f1 = be.array(np.ones(n, np.float32))
    runs1 = np.array([(0, M, n - 1, rank)], np.int32)
    C = be.array(c.c0)
    c.adapters = n
    c.call(be, X, *far, f1, be.rows_list(runs1), 1, C, True)
    want, tol = orc.lora(c.x, c.A[1:], c.B[1:], None, [(0, M, 0, rank)], c.c0, True)
    assert np.all(np.abs(C.download() - want) <= tol)
    [f.free() for f in far]


@gpu
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows,K", [([200, 100], 256), ([1, 1, 1], 256), ([1, 1, 1], 1280)])
def test_captured_with_infinities(be, orc, types, rows, K):
    """Replayed with an infinity in another row each time, the direct call between the replays."""
    c = Case(orc, sum(rows), 300, K, 16, 3, types, seed=1600)
    runs = np.array(ragged(rows, 3, 16), np.int32)
    X, A, B, scale = c.device(be)
    C, seg = be.array(c.c0), be.rows_list(runs)
    c.call(be, X, A, B, scale, seg, len(rows), C, True)
    be.capture_begin()
    c.call(be, X, A, B, scale, seg, len(rows), C, True)
    g = be.capture_end()
    clean = c.x.copy()
    try:
        for rep in range(4):
            c.x = clean.copy()
            c.x[rep * 7 % len(c.x), 5] = np.inf if rep else 1.0
            X.upload(f32_to_bf16(c.x) if types.startswith("bf16") else c.x)
            C.upload(c.c0)
            be.graph_launch(g)
            got = C.download()
            with np.errstate(invalid="ignore"):
                want, tol = orc.lora(c.x, c.A, c.B, c.scale, runs, c.c0, True)
            fin = np.isfinite(want)
            assert np.array_equal(np.isfinite(got), fin) and np.all(np.abs(got[fin] - want[fin]) <= tol[fin]), rep
            C.upload(c.c0)
            c.call(be, X, A, B, scale, seg, len(rows), C, True)
            assert np.array_equal(C.download().view(np.uint32), got.view(np.uint32)), rep
    finally:
        be.graph_destroy(g)
