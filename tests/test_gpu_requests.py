"""GPU test of the operators for batches of requests as a text model's layer uses them:
rows of ragged prompts through norm, shared projections, each request's adapter, rotary
positions and packed attention into a cache in slots, then single tokens against that
cache; directly and from two captured graphs. Every step is held to its own definition
in float64, from what the device had in hand before it."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SLOT = 96


def bf16(a):
    from oracle import f32_to_bf16 as f

    return f(a).reshape(np.shape(a))


def bf16_value(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Layer:
    dim, heads, kv, d, rank, adapters, eps = 256, 8, 2, 64, 8, 3, 1e-6

    def __init__(self, be, orc, requests, rows):
        self.be, self.orc, self.n = be, orc, requests
        hd, kd = self.heads * self.d, self.kv * self.d
        shapes = {"q": (hd, self.dim), "k": (kd, self.dim), "v": (kd, self.dim), "o": (self.dim, hd)}
        self.W = {n: bf16(orc.randn(s, 50 + i, 0.0, s[1] ** -0.5)) for i, (n, s) in enumerate(shapes.items())}
        self.A = {n: bf16(orc.randn((self.adapters, self.rank, shapes[n][1]), 60 + i, 0.0, shapes[n][1] ** -0.5))
                  for i, n in enumerate("qo")}
        self.B = {n: bf16(orc.randn((self.adapters, shapes[n][0], self.rank), 70 + i, 0.0, 0.5)) for i, n in enumerate("qo")}
        self.alpha = orc.randn((self.adapters,), 80)
        self.gamma = {n: orc.randn((s,), 81 + i, 1.0, 0.1) for i, (n, s) in
                      enumerate({"x": self.dim, "q": self.d, "k": self.d}.items())}
        self.dev = {n + w: be.array(a) for n, g in (("W", self.W), ("A", self.A), ("B", self.B), ("g", self.gamma))
                    for w, a in g.items()}
        self.dev["alpha"] = be.array(self.alpha)
        self.cache = {n: be.array(np.full((requests * SLOT, kd), np.nan, np.float32)) for n in "kv"}
        self.buf = {"x": be.empty((rows, self.dim)), "h": be.empty((rows, self.dim)),
                    "h16": be.array(np.zeros((rows, self.dim), np.uint16)), "q": be.empty((rows, hd)),
                    "k": be.empty((rows, kd)), "v": be.empty((rows, kd)), "a16": be.array(np.zeros((rows, hd), np.uint16)),
                    "cos": be.empty((rows, self.d)), "sin": be.empty((rows, self.d)),
                    "spans": be.rows_list(np.zeros((requests, 4), np.int32)),
                    "runs": be.rows_list(np.zeros((requests, 4), np.int32))}

    def set(self, x, lens, past):
        """The step's rows, lens[i] of request i behind past[i] keys."""
        first = np.cumsum([0] + list(lens))
        self.T, self.lens, self.past = int(first[-1]), list(lens), list(past)
        self.spans = np.array([(first[i], n, i * SLOT, past[i] + n) for i, n in enumerate(lens)], np.int32)
        self.runs = np.array([(first[i], n, i % (self.adapters + 1) - 1, self.rank - i % 2) for i, n in enumerate(lens)], np.int32)
        at = np.concatenate([past[i] + np.arange(n) for i, n in enumerate(lens)])[:, None] / 100.0 ** (np.arange(self.d) % 32 / 32)
        self.cos, self.sin = np.cos(at).astype(np.float32), np.sin(at).astype(np.float32)
        for n, a in (("x", x), ("cos", self.cos), ("sin", self.sin), ("spans", self.spans), ("runs", self.runs)):
            self.be.upload(self.buf[n].ptr, np.ascontiguousarray(a))

    def project(self):
        be, b, w, T, hd, kd = self.be, self.buf, self.dev, self.T, self.heads * self.d, self.kv * self.d
        be.rms_norm(b["x"], b["h"], T, self.dim, w["gx"], self.eps)
        be.to_bf16(b["h"], b["h16"], T * self.dim)
        for n, N in (("q", hd), ("k", kd), ("v", kd)):
            be.gemm_nt_bf16_packed(T, N, self.dim, b["h16"], self.dim, w["W" + n], self.dim, b[n], N)
        be.lora_nt_bf16_packed(T, hd, self.dim, b["h16"], self.dim, w["Aq"], w["Bq"], self.rank, self.adapters, w["alpha"],
                               b["runs"], self.n, b["q"], hd)

    def rotate(self):
        b, w = self.buf, self.dev
        self.be.qknorm_rope(b["q"], self.heads * self.d, b["k"], self.kv * self.d, 1, self.T, self.d, w["gq"], w["gk"],
                            self.eps, b["cos"], b["sin"], False)

    def store(self):
        kd = self.kv * self.d * 4
        for (q0, n, k0, _), past in zip(self.spans.tolist(), self.past):
            for c in "kv":
                self.be.copy(self.cache[c].ptr + (k0 + past) * kd, self.buf[c].ptr + q0 * kd, n * kd)

    def attend(self):
        be, b, w, T, hd = self.be, self.buf, self.dev, self.T, self.heads * self.d
        be.attention_packed(b["q"], self.cache["k"], self.cache["v"], b["a16"], T, self.n * SLOT, self.heads, self.kv, self.d,
                            b["spans"], self.n, self.d ** -0.5, causal=True, out_bf16=True)
        be.gemm_nt_bf16_packed(T, self.dim, hd, b["a16"], hd, w["Wo"], hd, b["x"], self.dim, None, True)
        be.lora_nt_bf16_packed(T, self.dim, hd, b["a16"], hd, w["Ao"], w["Bo"], self.rank, self.adapters, w["alpha"],
                               b["runs"], self.n, b["x"], self.dim)

    def get(self, n):
        a = self.buf[n].download()[:self.T]
        return bf16_value(a) if n.endswith("16") else a

    def projected(self, n, x16, c0=0.0):
        """x16 W^T (+ the adapters') from c0, and its bound."""
        W = bf16_value(self.W[n]).astype(np.float64)
        base = c0 + x16.astype(np.float64) @ W.T
        tol = (x16.shape[1] + 4) * U * (np.abs(x16).astype(np.float64) @ np.abs(W).T + np.abs(c0))
        if n not in self.A:
            return base, tol
        want, more = self.orc.lora(x16, bf16_value(self.A[n]), bf16_value(self.B[n]), self.alpha, self.runs, base, True)
        return want, tol + more

    def checked(self, what):
        """The step, every stage against its definition."""
        def near(got, want, tol, name):
            over = np.abs(got - want) - tol
            assert np.all(over <= 0), f"{what} {name}: {np.nanmax(over):.3e} beyond the bound"

        x = self.get("x")
        self.project()
        h = x.astype(np.float64)
        h = h / np.sqrt(np.mean(h * h, -1, keepdims=True) + self.eps) * self.gamma["x"]
        near(self.get("h16"), h, np.abs(h) * (2.0 ** -8 + (self.dim + 16) * U), "norm")
        for n in "qkv":
            near(self.get(n), *self.projected(n, self.get("h16")), n)
        before = {n: self.get(n) for n in "qk"}
        self.rotate()
        for n in "qk":
            a = before[n].astype(np.float64).reshape(self.T, -1, self.d)
            a = a / np.sqrt(np.mean(a * a, -1, keepdims=True) + self.eps) * self.gamma[n]
            half = self.d // 2
            turned = np.concatenate((-a[..., half:], a[..., :half]), -1)
            c, s = self.cos[:, None, :], self.sin[:, None, :]
            near(self.get(n).reshape(a.shape), a * c + turned * s, (self.d + 24) * U * (np.abs(a * c) + np.abs(turned * s)), "rotated " + n)
        self.store()
        self.attend()
        k, v = self.cache["k"].download(), self.cache["v"].download()
        for (q0, n, k0, _), past in zip(self.spans.tolist(), self.past):
            assert np.array_equal(k[k0 + past:k0 + past + n], self.get("k")[q0:q0 + n])
        want, tol = self.orc.attention_packed(self.get("q"), k, v, np.zeros((self.T, self.heads * self.d)), self.spans, self.heads,
                                              self.kv, self.d ** -0.5, causal=True)
        near(self.get("a16"), want, tol + 2.0 ** -8 * (np.abs(want) + tol), "attention")
        near(self.get("x"), *self.projected("o", self.get("a16"), x), "out")
        assert np.all(np.isfinite(self.get("x"))), what


@pytest.mark.parametrize("lens", [[5, 33, 1, 77, 20], [1], [64, 64]], ids=str)
def test_prompts_then_tokens(be, orc, lens):
    """The cache starts as NaN: rows behind a request's keys are in its slot, not in its results."""
    L = Layer(be, orc, len(lens), sum(lens))
    L.set(orc.randn((sum(lens), L.dim), 1), lens, [0] * len(lens))
    L.checked("prompts")
    for step in range(3):
        past = [n + step for n in lens]
        L.set(orc.randn((len(lens), L.dim), 2 + step), [1] * len(lens), past)
        L.checked(f"token {step}")


def test_tokens_from_graphs(be, orc):
    """A step's two halves as graphs, replayed with other rows, positions and lengths, the same
    step called directly between the replays: the same bits."""
    lens = [5, 33, 1, 77, 20]
    L = Layer(be, orc, len(lens), sum(lens))
    L.set(orc.randn((sum(lens), L.dim), 1), lens, [0] * len(lens))
    L.checked("prompts")

    def step(i, first, second):
        L.set(orc.randn((len(lens), L.dim), 20 + i), [1] * len(lens), [n + i for n in lens])
        first()
        L.store()
        second()
        return L.get("x"), L.cache["k"].download(), L.cache["v"].download()

    def first():
        L.project()
        L.rotate()

    step(0, first, L.attend)
    graphs = []
    try:
        for half in (first, L.attend):
            be.capture_begin()
            half()
            graphs.append(be.capture_end())
        for i in range(4):
            direct = step(i, first, L.attend)
            replayed = step(i, *(lambda g=g: be.graph_launch(g) for g in graphs))
            for a, b in zip(direct, replayed):
                assert np.array_equal(a, b, equal_nan=True), i
    finally:
        for g in graphs:
            be.graph_destroy(g)


HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
FRESH = r"""
import sys
sys.path[:0] = [%r, %r]
import numpy as np, sdhip
from oracle import Oracle
be, orc = sdhip.Backend(), Oracle()
T, heads, d = 200, 4, 64
q, k, v = (be.array(orc.randn((T, heads * d), i)) for i in range(3))
out, spans = be.empty((T, heads * d)), np.array([(0, 150, 0, 150), (150, 50, 150, 50)], np.int32)
dspans = be.rows_list(spans)
X, A, B, C = be.array(orc.randn((T, 1280), 4)), orc.randn((2, 8, 1280), 5, 0.0, 0.03), orc.randn((2, 96, 8), 6), be.array(np.zeros((T, 96), np.float32))
dA, dB, runs = be.array(A), be.array(B), np.array([(0, 150, 0, 8), (150, 50, 1, 8)], np.int32)
druns = be.rows_list(runs)
def attend():
    be.attention_packed(q, k, v, out, T, T, heads, heads, d, dspans, 2, 0.125, causal=True)
def adapt():
    be.lora_nt_f32(T, 96, 1280, X, 1280, dA, dB, 8, 2, None, druns, 2, C, 96, accumulate=False)
be.capture_begin()
attend()
try:
    adapt()
    raise SystemExit('not refused')
except sdhip.SdhError as e:
    assert e.status == sdhip.SDH_ERR_INVALID and 'captur' in str(e), e
graph = be.capture_end()
adapt()
be.capture_begin()
adapt()
second = be.capture_end()
for i in range(3):
    x = orc.randn((T, heads * d), 10 + i)
    q.upload(x)
    be.call('sdh_zero', out.ptr, out.nbytes)
    be.call('sdh_zero', C.ptr, C.nbytes)
    be.graph_launch(graph)
    be.graph_launch(second)
    want, tol = orc.attention_packed(x, k.download(), v.download(), np.zeros((T, heads * d)), spans, heads, heads, 0.125, causal=True)
    assert np.all(np.abs(out.download() - want) <= tol), i
    want, tol = orc.lora(X.download(), A, B, None, runs, np.zeros((T, 96)), False)
    assert np.all(np.abs(C.download() - want) <= tol), i
    attend()
    adapt()
    be.synchronize()
be.graph_destroy(graph)
be.graph_destroy(second)
print('fresh ok', flush=True)
""" % (os.path.join(ROOT, "stablediffusion-cpp_amd"), os.path.join(ROOT, "oracle"))


def test_captured_before_any_call():
    """In a process where no call has had scratch: attention goes without, the adapters are refused until they have run."""
    r = subprocess.run([sys.executable, "-u", "-c", FRESH], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr[-3000:])
    assert r.returncode == 0 and "fresh ok" in r.stdout
