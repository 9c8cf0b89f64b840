"""GPU tests of low-rank adapters (sdh_lora_nt_*) at infinities, against the float64
definition (Oracle.lora)."""
import numpy as np
import pytest

from test_gpu_lora import TYPES, Case, bf16_value, f32_to_bf16

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
