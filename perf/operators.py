"""Measurable cases of the operators for batches of requests: attention over packed sequences, and low-rank adapters.

A program that serves many requests keeps their rows in one tensor, one request after another, and says in an int32
array which rows are whose. Two operators work on such tensors:

  attention   sdhip.Backend.attention_packed: every sequence's queries attend that sequence's keys, under a causal,
              window or prefix mask, with scores capped by a tanh or biased by distance.
  lora        sdhip.Backend.lora_nt_*: C += scale_a (X A_a^T) B_a^T, each run of rows with the adapter a of its own
              request, beside a projection that all of them share.

With own false, run() computes them from elementary torch operations in fp32; with own true it calls the library,
which works on a stream of its own: prepare() returns once the inputs are there, and a program waits for the device
(torch.cuda.synchronize(), Backend.synchronize()) before torch reads what run() returned.
listed() and draw() give the cases, prepare() what a program has in hand, work() what a pass has to move and compute,
exact() the results in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------- the cases
# seqs sequences (or runs of rows) of min_len to max_len rows; `lens` seeds their lengths.
def _attention(name, **kw):
    c = {"name": name, "kind": "attention", "seqs": 1, "q_len": 0, "min_len": 1, "max_len": 1, "slots": False,
         "heads": 8, "kv_heads": 8, "d": 64, "causal": True, "window": 0, "prefix": 0, "cap": 0.0, "radius": 0,
         "out_bf16": False, "lens": 1}
    c.update(kw)
    return c


def _lora(name, **kw):
    c = {"name": name, "kind": "lora", "seqs": 1, "min_len": 1, "max_len": 1, "K": 256, "N": 256, "rank": 16,
         "adapters": 4, "types": "f32_bf16", "accumulate": True, "lens": 1}
    c.update(kw)
    return c


def listed():
    return [
        # the adaLN modulation of four requests' timesteps: one row each; the smallest call, where latency counts
        _lora("lora_modulation", seqs=4, K=256, N=15360, rank=8),
        # one token of each of 48 requests through a text model's query projection
        _lora("lora_tokens", seqs=48, K=2560, N=4096, rank=16, adapters=24, types="bf16_bf16"),
        # ragged prompts through the same projection, adapters of up to 32 ranks
        _lora("lora_prompts", seqs=24, min_len=5, max_len=203, K=2560, N=4096, rank=32, adapters=10),
        # fp32 adapters on a UNet's feed-forward front, eight latents of 32 x 32 pixels
        _lora("lora_unet", seqs=8, min_len=1024, max_len=1024, K=640, N=5120, rank=12, types="f32_f32"),
        # image + text rows of three images through a DiT's feed-forward front, written ahead of the shared product
        _lora("lora_images", seqs=3, min_len=4128, max_len=4224, K=3840, N=10240, rank=64, types="bf16_bf16",
              accumulate=False),
        # CLIP prompts, padded to 77 tokens each in the batch, of which the real ones count
        _attention("attention_clip", seqs=16, min_len=5, max_len=77, slots=True, heads=12, kv_heads=12, d=64),
        # ragged prompts of a text model with grouped heads
        _attention("attention_prompts", seqs=24, min_len=5, max_len=203, heads=32, kv_heads=8, d=128),
        # one new token per request against its cached keys, in slots of 4096
        _attention("attention_tokens", seqs=32, q_len=1, min_len=40, max_len=4096, slots=True, heads=32, kv_heads=8,
                   d=128),
        # one request's token against a long cache
        _attention("attention_token_long", seqs=1, q_len=1, min_len=30001, max_len=30001, heads=32, kv_heads=8,
                   d=128),
        # an encoder with a bias by distance (clamped at 128), both directions
        _attention("attention_distance", seqs=12, min_len=77, max_len=512, heads=24, kv_heads=24, d=64, causal=False,
                   radius=128),
        # long prompts: capped scores, a window, a prefix that all rows see
        _attention("attention_window", seqs=4, min_len=1500, max_len=2400, heads=16, kv_heads=4, d=128, window=512,
                   prefix=64, cap=50.0, out_bf16=True),
        # image + text sequences of two images, all rows to all rows of their own image; the largest
        _attention("attention_images", seqs=2, min_len=4128, max_len=4224, heads=30, kv_heads=30, d=128,
                   causal=False, out_bf16=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    lens = rng.randrange(1, 1 << 30)
    if rng.random() < 0.4:
        seqs = _log(rng, 1, 64)
        top = _log(rng, 1, max(1, 8448 // seqs))
        c = _lora("", seqs=seqs, min_len=rng.randrange(top) + 1, max_len=top, lens=lens,
                  K=rng.choice((256, 320, 640, 650, 1280, 2560, 3840)),
                  N=rng.choice((320, 1000, 1885, 2560, 4096, 5120, 9728, 10240)),
                  rank=rng.choice((4, 8, 12, 16, 21, 32, 64, 128)), adapters=rng.randrange(seqs) + 1,
                  types=rng.choice(("f32_bf16", "bf16_bf16", "f32_f32")), accumulate=rng.random() < 0.7)
    elif rng.random() < 0.4:
        seqs = _log(rng, 1, 64)
        top = _log(rng, 16, 131072 // seqs)
        heads, kv = rng.choice(((32, 8), (16, 4), (12, 12), (8, 1), (30, 30)))
        c = _attention("", seqs=seqs, q_len=rng.choice((1, 1, 1, 2, 5)), min_len=max(5, rng.randrange(top)),
                       max_len=max(5, top), slots=rng.random() < 0.5, heads=heads, kv_heads=kv,
                       d=rng.choice((64, 128)), window=rng.choice((0, 0, 1024)), cap=rng.choice((0.0, 30.0)),
                       lens=lens)
    else:
        seqs = _log(rng, 1, 32)
        top = _log(rng, 5, min(4224, 8448 // seqs))
        heads, kv, d = rng.choice(((32, 8, 128), (12, 12, 64), (16, 16, 64), (30, 30, 128), (8, 8, 40), (8, 8, 80),
                                   (8, 2, 96)))
        causal = rng.random() < 0.6
        c = _attention("", seqs=seqs, min_len=rng.randrange(top) + 1, max_len=top, heads=heads, kv_heads=kv, d=d,
                       causal=causal, window=rng.choice((0, 0, 7, 256)), prefix=rng.choice((0, 0, 9, 100)),
                       cap=rng.choice((0.0, 0.0, 50.0)), radius=rng.choice((0, 0, 128)),
                       out_bf16=rng.random() < 0.3, slots=rng.random() < 0.3, lens=lens)
    del c["name"]
    return c


def _rows(c):
    """The case's sequences as (first row, rows) of queries and of keys, the rows of both tensors, and a generator for the rest."""
    g = random.Random(c["lens"])
    n = [g.randint(c["min_len"], c["max_len"]) for _ in range(c["seqs"])]
    if c["kind"] == "lora" or not c["slots"]:
        first = [sum(n[:i]) for i in range(len(n))]
        keys, Tk = list(zip(first, n)), sum(n)
    else:
        keys, Tk = [(i * c["max_len"], m) for i, m in enumerate(n)], c["seqs"] * c["max_len"]
    if c["kind"] == "attention" and c["q_len"]:
        return [(i * c["q_len"], c["q_len"]) for i in range(len(n))], keys, c["seqs"] * c["q_len"], Tk, g
    return keys, keys, Tk, Tk, g


def _segments(c):
    """(first row, rows, adapter, rank) of each run of rows; some have no adapter."""
    rows, _, M, _, g = _rows(c)
    ranks = [c["rank"] if i == 0 else g.choice((c["rank"], c["rank"], (c["rank"] + 1) // 2)) for i in range(c["adapters"])]
    seg = []
    for i, (first, n) in enumerate(rows):
        a = i % c["adapters"] if i < c["adapters"] else g.randrange(-1, c["adapters"])
        seg.append((first, n, a, ranks[a] if a >= 0 else 0))
    return seg, M


def _prefixes(c):
    g = _rows(c)[4]
    return [g.randint(0, c["prefix"]) for _ in range(c["seqs"])]


# ---------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    st = {"case": c}
    if c["kind"] == "lora":
        seg, M = _segments(c)
        x, w = (torch.bfloat16 if t == "bf16" else torch.float32 for t in c["types"].split("_"))
        K, N, r, n = c["K"], c["N"], c["rank"], c["adapters"]
        # hidden rows have channels of unequal size; a trained adapter's two factors are alike in size
        st["x"] = (randn(M, K) * torch.exp(0.5 * randn(K))).to(x)
        st["A"] = randn(n, r, K, std=1 / math.sqrt(K), dtype=w)
        st["B"] = randn(n, N, r, std=0.3 / math.sqrt(r), dtype=w)
        st["scale"] = torch.rand(n, generator=g, device="cuda") + 0.5
        st["segments"] = ints(seg)
        st["y"] = randn(M, N) if c["accumulate"] else torch.zeros(M, N, device="cuda")
        torch.cuda.synchronize()  # the library works on a stream of its own
        return st
    q, k, Tq, Tk, _ = _rows(c)
    h, kv, d = c["heads"], c["kv_heads"], c["d"]
    st["q"], st["k"], st["v"] = randn(Tq, h * d, std=1.5), randn(Tk, kv * d), randn(Tk, kv * d)
    st["spans"] = ints([a + b for a, b in zip(q, k)])
    st["prefix"] = ints(_prefixes(c)) if c["prefix"] else None
    st["bias"] = randn(h, 2 * c["radius"] + 1) if c["radius"] else None
    st["out"] = torch.zeros(Tq, h * d, device="cuda", dtype=torch.bfloat16 if c["out_bf16"] else torch.float32)
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------------------ runs
def _lora_plain(st):
    """All runs of rows at once, padded to the longest."""
    c, x, y, seg = st["case"], st["x"], st["y"], st["segments"].long()
    first, n, a, rank = seg.unbind(1)
    i = torch.arange(c["max_len"], device="cuda")
    inside = i < n[:, None]
    at = (first[:, None] + i).clamp(max=x.shape[0] - 1)
    A = st["A"].float()[a.clamp(min=0)]
    B = st["B"].float()[a.clamp(min=0)]
    h = torch.matmul(x.float()[at], A.transpose(1, 2).contiguous())
    h = h * (torch.arange(c["rank"], device="cuda") < rank[:, None])[:, None, :]
    delta = torch.matmul(h, B.transpose(1, 2).contiguous()) * st["scale"][a.clamp(min=0)][:, None, None]
    rows = at[inside]
    y[rows] = y[rows] + delta[inside] if c["accumulate"] else delta[inside]
    return y


def _attention_plain(st):
    """All sequences at once, padded to the longest."""
    c, q, k, v, out = st["case"], st["q"], st["k"], st["v"], st["out"]
    h, kv, d = c["heads"], c["kv_heads"], c["d"]
    q0, lq, k0, lk = st["spans"].long().unbind(1)
    i = torch.arange(c["q_len"] or c["max_len"], device="cuda")
    j = torch.arange(c["max_len"], device="cuda")
    qi = (q0[:, None] + i).clamp(max=q.shape[0] - 1)
    kj = (k0[:, None] + j).clamp(max=k.shape[0] - 1)
    S, Lq, Lk = len(lq), len(i), len(j)
    qs = q[qi].reshape(S, Lq, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(S, kv, -1, d).contiguous()
    ks = k[kj].reshape(S, Lk, kv, d).permute(0, 2, 3, 1).contiguous()
    vs = v[kj].reshape(S, Lk, kv, d).permute(0, 2, 1, 3).contiguous()
    vs = torch.where((j < lk[:, None])[:, None, :, None], vs, 0.0)
    s = torch.matmul(qs, ks).reshape(S, h, Lq, Lk) / math.sqrt(d)
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    pos = i + (lk - lq)[:, None]  # a row's place among its sequence's keys: the last row stands at the last key
    dist = j - pos[:, :, None]
    if c["radius"]:
        s = s + st["bias"][:, dist.clamp(-c["radius"], c["radius"]) + c["radius"]].transpose(0, 1)
    seen = torch.ones_like(dist, dtype=torch.bool)
    if c["causal"]:
        seen &= dist <= 0
    if c["window"]:
        seen &= dist.abs() < c["window"]
    if c["prefix"]:
        seen |= j < st["prefix"].long()[:, None, None]
    seen &= j < lk[:, None, None]
    s = torch.where(seen[:, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p.reshape(S, kv, -1, Lk), vs).reshape(S, h, Lq, d).transpose(1, 2).reshape(S, Lq, h * d)
    inside = i < lq[:, None]
    out[qi[inside]] = o[inside].to(out.dtype)
    return out


class _Known:
    """A state's tensors, known to the library for as long as the state lives."""

    def __init__(self, st):
        sys.path.insert(0, os.path.join(ROOT, "stablediffusion-cpp_amd"))
        import sdhip

        _Known.be = getattr(_Known, "be", None) or sdhip.Backend()
        self.ptr = {n: t.data_ptr() for n, t in st.items() if isinstance(t, torch.Tensor)}
        for n, p in self.ptr.items():
            self.be.register_external(p, st[n].numel() * st[n].element_size())

    def __del__(self):
        for p in self.ptr.values():
            self.be.unregister_external(p)


def run(state):
    c = state["case"]
    if not own:
        return _lora_plain(state) if c["kind"] == "lora" else _attention_plain(state)
    known = state.get("known") or state.setdefault("known", _Known(state))
    be, p = known.be, known.ptr
    if c["kind"] == "lora":
        call = {"f32_bf16": be.lora_nt_bf16, "bf16_bf16": be.lora_nt_bf16_packed, "f32_f32": be.lora_nt_f32}
        call[c["types"]](state["x"].shape[0], c["N"], c["K"], p["x"], c["K"], p["A"], p["B"], c["rank"],
                         c["adapters"], p["scale"], p["segments"], c["seqs"], p["y"], c["N"],
                         accumulate=c["accumulate"])
        return state["y"]
    be.attention_packed(p["q"], p["k"], p["v"], p["out"], state["q"].shape[0], state["k"].shape[0], c["heads"],
                        c["kv_heads"], c["d"], p["spans"], c["seqs"], 1 / math.sqrt(c["d"]), causal=c["causal"],
                        window=c["window"], prefix=p.get("prefix"), cap=c["cap"], bias=p.get("bias"),
                        radius=c["radius"], out_bf16=c["out_bf16"])
    return state["out"]


# ------------------------------------------------------------ what a pass needs
def _seen(c, lq, lk, prefix):
    """How many keys each row of a sequence sees, as a list, and how many keys any of them sees."""
    w = c["window"]
    seen, keys = [], set()
    for i in range(lq):
        p = i + lk - lq
        lo = max(0, p - w + 1) if w else 0
        hi = min(lk, p + 1 if c["causal"] else p + w if w else lk)
        lo, hi = min(lo, lk), max(hi, 0)
        a = min(prefix, lk)
        seen.append(max(0, hi - max(lo, a)) + a)
        keys.add((max(lo, a), max(hi, max(lo, a))))
    low, high = min(x for x, _ in keys), max(y for _, y in keys)
    return seen, min(prefix, lk) + max(0, high - low)


def work(c):
    if c["kind"] == "lora":
        seg, M = _segments(c)
        tx, tw = (2 if t == "bf16" else 4 for t in c["types"].split("_"))
        rows = sum(n for _, n, a, r in seg if a >= 0 and r)
        used = {a: r for _, n, a, r in seg if a >= 0 and n}
        moved = rows * c["K"] * tx + rows * c["N"] * 4 * (2 if c["accumulate"] else 1)
        if not c["accumulate"]:
            moved += (sum(n for _, n, _, _ in seg) - rows) * c["N"] * 4
        moved += sum(r * (c["K"] + c["N"]) * tw + 4 for r in used.values()) + 16 * len(seg)
        return {"bytes": moved, "flops": sum(2 * n * r * (c["K"] + c["N"]) for _, n, _, r in seg)}
    q, k, _, _, _ = _rows(c)
    prefix = _prefixes(c)
    pairs = keys = 0
    for (_, lq), (_, lk), p in zip(q, k, prefix):
        s, n = _seen(c, lq, lk, p)
        pairs, keys = pairs + sum(s), keys + n
    rows = sum(n for _, n in q)
    moved = rows * c["heads"] * c["d"] * (6 if c["out_bf16"] else 8) + keys * c["kv_heads"] * c["d"] * 8
    moved += c["heads"] * (2 * c["radius"] + 1) * 4 * (c["radius"] > 0) + 16 * c["seqs"]
    return {"bytes": moved, "flops": 4 * pairs * c["heads"] * c["d"]}


# --------------------------------------------------------------------- 64 bits
def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] == "lora":
        y = st["y"].double()
        for first, n, a, r in _segments(c)[0]:
            to = slice(first, first + n)
            if not c["accumulate"]:
                y[to] = 0
            if a >= 0 and n and r:
                h = st["x"][to].double() @ st["A"][a, :r].double().t().contiguous()
                y[to] += st["scale"][a].double() * (h @ st["B"][a, :, :r].double().t().contiguous())
        return y
    q, k, _, _, _ = _rows(c)
    h, group, d = c["heads"], c["heads"] // c["kv_heads"], c["d"]
    out = st["out"].double()
    for (q0, lq), (k0, lk), pre in zip(q, k, _prefixes(c)):
        if not lq or not lk:
            continue
        at = torch.arange(lk - lq, lk, device="cuda").unsqueeze(1) - torch.arange(lk, device="cuda")
        hidden = torch.zeros(lq, lk, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden = at < 0
        if c["window"]:
            hidden = hidden | (at >= c["window"]) | (at <= -c["window"])
        hidden[:, :pre] = False
        empty = hidden.all(1)
        for n in range(h):
            f = slice(n * d, n * d + d)
            g = slice(n // group * d, n // group * d + d)
            s = st["q"][q0:q0 + lq, f].double() @ st["k"][k0:k0 + lk, g].double().t().contiguous() / math.sqrt(d)
            if c["cap"]:
                s = torch.tanh(s / c["cap"]) * c["cap"]
            if c["radius"]:
                s = s + st["bias"][n].double()[c["radius"] - at.clamp(-c["radius"], c["radius"])]
            s = torch.softmax(s.masked_fill(hidden, -math.inf), 1).masked_fill(empty[:, None], 0.0)
            out[q0:q0 + lq, f] = s @ st["v"][k0:k0 + lk, g].double()
    return out
