"""GPU tests of a decoder layer of a batch of sessions from the standalone operators, as a server runs it: rows
normalised and quantised, products on 8-bit integers, queries and keys rotated and stored, attention over pages (whole,
windowed, or with a shared prefix), and the residuals; eagerly, captured into graphs, and on two streams."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_forms_ref as forms  # noqa: E402
import paged_ref as ref  # noqa: E402
from instantcua_amd import engine as eng  # noqa: E402
from instantcua_amd import int8, paged  # noqa: E402
from instantcua_amd.modelfile import WeightFormat  # noqa: E402
from test_gpu_int8 import check as check_product, product, quantised  # noqa: E402
from test_gpu_paged import D, dev, download, tables_of, upload  # noqa: E402
from test_gpu_paged_use import Hip, put  # noqa: E402

pytestmark = pytest.mark.gpu
H, HEADS, KV, FF, PAGE = 512, 4, 2, 784, 16
F32, F16 = paged.F32, paged.F16
EPS = 1e-6


class Layer:
    """Weights, a cache with room for `lens` slots a session, and buffers for up to `tokens` new tokens, all at fixed
    addresses.  Sessions 0 .. shared - 1 have the first `prefix` slots in common; `window` (slots, first ones)."""

    def __init__(self, fmt, lens, tokens, shared=0, prefix=0, window=None, seed=0):
        rng = np.random.default_rng(seed)
        self.rng, self.lens, self.tokens, self.shared, self.prefix, self.window = rng, lens, tokens, shared, prefix, window
        self.weights = {}
        for name, (n, k) in {"qkv": ((HEADS + 2 * KV) * D, H), "o": (H, HEADS * D), "gate_up": (2 * FF, H), "down": (H, FF)}.items():
            w = dev((rng.standard_normal((n, k)) / k ** 0.5).astype(np.float32))
            codes, scales = eng.DeviceBuffer(n * k), eng.DeviceBuffer(4 * n)
            int8.quantize(w, codes, scales, n, k)  # a matrix: each channel is a row
            self.weights[name] = (codes, scales, n, k)
        self.norms = {k: dev((1 + 0.2 * rng.standard_normal(n)).astype(np.float32)) for k, n in (("in", H), ("ff", H), ("q", D), ("k", D))}
        self.table, pages = tables_of(lens, PAGE, rng)
        for s in range(1, shared):
            self.table[s, :prefix // PAGE] = self.table[0, :prefix // PAGE]
        self.pool = ref.Pool(fmt, KV, PAGE, pages)
        for s in range(len(lens)):  # what the sessions had before
            p = np.arange(lens[s])
            self.pool.fill(self.table[s, p // PAGE].astype(np.int64) * PAGE + p % PAGE, rng)
        self.cache = upload(self.pool)
        self.rope = dev(ref.rope_table(max(lens), D))
        self.b = {k: eng.DeviceBuffer(tokens * n) for k, n in {
            "x": 4 * H, "codes": 1024, "scales": 4, "qkv": 4 * (HEADS + 2 * KV) * D, "q": 2 * HEADS * D, "attn": 2 * HEADS * D,
            "mid": 4 * H, "h": 2 * FF, "out": 4 * H, "pos": 4, "slots": 4}.items()}
        self.start, self.kv, self.tables = eng.DeviceBuffer(4 * (len(lens) + 1)), eng.DeviceBuffer(4 * len(lens)), dev(self.table)
        self.groups = [dev(np.array(a, np.int32)) for a in ([0, shared], [prefix])]
        self.sizes = dict(max_q=tokens, max_kv=max(lens))
        args = (HEADS, len(lens), tokens)
        c = self.cache
        need = (c.attention_window_work(*args, *window, **self.sizes) if window else
                c.attention_prefix_work(*args, 1, prefix, **self.sizes) if prefix else c.attention_work(*args, **self.sizes))
        self.work = eng.DeviceBuffer(need) if need else None

    def load(self, news, have):
        """New tokens' rows, and where they go: session s has have[s] slots before its news[s] new ones; rows behind
        the last session's have no slot."""
        T = sum(news)
        self.news, self.have = news, [h + n for h, n in zip(have, news)]
        x = np.zeros((self.tokens, H), np.float32)
        x[:T] = self.rng.standard_normal((T, H)) * 2
        pos, slots = np.zeros(self.tokens, np.int32), np.full(self.tokens, -1, np.int32)
        pos[:T] = np.concatenate([np.arange(h, h + n) for h, n in zip(have, news)])
        slots[:T] = np.concatenate([self.cache.slots(t, h, n) for t, h, n in zip(self.table, have, news)])
        self.slots = slots[:T]
        for b, a in ((self.b["x"], x), (self.b["pos"], pos), (self.b["slots"], slots), (self.kv, np.array(self.have, np.int32)),
                     (self.start, np.concatenate([[0], np.cumsum(news)]).astype(np.int32))):
            put(b, a)

    def product(self, src, src_type, name, y, y_type, norm=None, add=None, stream=0):
        codes, scales, n, k = self.weights[name]
        b, gated = self.b, name == "gate_up"
        int8.quantize(b[src], b["codes"], b["scales"], self.tokens, k, norm=norm, eps=EPS, type=src_type, stream=stream)
        int8.matmul(b["codes"], b["scales"], codes, scales, b[y], self.tokens, n // 2 if gated else n, k,
                    add=None if add is None else b[add], gated=gated, type=y_type, stream=stream)

    def enqueue(self, stream=0):
        b, c = self.b, self.cache
        self.product("x", F32, "qkv", "qkv", F32, norm=self.norms["in"], stream=stream)
        c.store(b["qkv"], self.tokens, b["slots"], n_heads=HEADS, q=b["q"], q_norm=self.norms["q"], k_norm=self.norms["k"],
                rope=self.rope, rope_rows=max(self.lens), pos=b["pos"], q_type=F16, stream=stream)
        args = (b["q"], b["attn"], HEADS, self.start, self.kv, self.tables, len(self.lens), self.tokens, self.table.shape[1])
        more = dict(type=F16, work=self.work, stream=stream, **self.sizes)
        if self.window:
            c.attention_window(*args, *self.window, **more)
        elif self.prefix:
            c.attention_prefix(*args, *self.groups, 1, self.prefix, **more)
        else:
            c.attention(*args, **more)
        self.product("attn", F16, "o", "mid", F32, add="x", stream=stream)
        self.product("mid", F32, "gate_up", "h", F16, norm=self.norms["ff"], stream=stream)
        self.product("h", F16, "down", "out", F32, add="mid", stream=stream)

    def get(self, name, dtype, width):
        return self.b[name].to_array(dtype, (self.tokens, width))[:sum(self.news)]

    def check(self):
        """Every operator's outputs against its definition on what it was given."""
        x, qkv = self.get("x", np.float32, H), self.get("qkv", np.float32, (HEADS + 2 * KV) * D)
        q, attn = (self.get(k, np.float16, HEADS * D) for k in ("q", "attn"))
        mid, h, out = self.get("mid", np.float32, H), self.get("h", np.float16, FF), self.get("out", np.float32, H)

        def of_product(src, name, got, type_, norm=None, add=None):
            codes, scales, n, k = self.weights[name]
            xc, xs = quantised(src, norm if norm is None else norm.to_array(np.float32, k))
            w, ws = codes.to_array(np.int8, (n, k)), scales.to_array(np.float32, n)
            want, tol = product(xc, xs.astype(np.float32), w, ws, add, name == "gate_up")
            # The scales of rows are the definition's to one step of fp32 more than rounding it.
            check_product(got, want, tol + 2.0 ** -23 * np.abs(want - (0 if add is None else add)) * (2 + np.abs(want)), type_)

        of_product(x, "qkv", qkv, F32, self.norms["in"])
        pool = download(self.cache, self.pool)
        group, T = HEADS // KV, sum(self.news)
        qd = q.astype(np.float64).reshape(T, HEADS, D)
        want, reach, vmax = forms.attention(pool, qd, self.news, self.have, self.table, *(self.window or (None, 0)))
        assert np.abs(attn.reshape(T, HEADS, D) - want).max() <= ref.attention_tol(True, pool.q8, reach, vmax) and group == 2
        of_product(attn, "o", mid, F32, add=x)
        of_product(mid, "gate_up", h, F16, self.norms["ff"])
        of_product(h, "down", out, F32, add=mid)
        return out


FORMS = {"whole": {}, "window": {"window": (37, 3)}, "prefix": {"shared": 3, "prefix": 160}}
LENS = (300, 290, 200, 260)
STEPS = [((1, 1, 1, 1), (250, 200, 160, 100)), ((3, 0, 20, 1), (251, 201, 161, 101)), ((1, 40, 1, 1), (254, 201, 181, 102)),
         ((1, 1, 1, 0), (255, 241, 182, 103))]


@pytest.mark.parametrize("fmt", [WeightFormat.F16, WeightFormat.Q8])
@pytest.mark.parametrize("form", list(FORMS))
def test_a_layer(fmt, form):
    layer = Layer(fmt, LENS, 48, **FORMS[form])
    for news, have in STEPS:
        layer.load(news, have)
        layer.enqueue()
        layer.check()


@pytest.mark.parametrize("form", list(FORMS))
def test_a_captured_layer_replays_with_new_tokens(form):
    """Captured once; the replays have other tokens, lengths and positions, among eager work and waits.  Each is the
    eager layer's to the bit."""
    hip = Hip()
    stream = hip.stream()
    layer, eager = (Layer(WeightFormat.F16, LENS, 48, seed=3, **FORMS[form]) for _ in range(2))
    ready = None
    for news, have in STEPS + STEPS[:2]:
        for e in (layer, eager):
            e.load(news, have)
        if ready is None:
            ready = hip.capture(stream, layer.enqueue)
        hip.call("hipGraphLaunch", ready, stream)
        hip.call("hipStreamSynchronize", stream)
        eager.enqueue()
        assert np.array_equal(layer.get("out", np.float32, H), eager.check())
    hip.call("hipGraphExecDestroy", ready)
    hip.call("hipStreamDestroy", stream)


def test_layers_on_two_streams():
    """Two batches at once, each with its own buffers: what each gives alone."""
    hip = Hip()
    streams = [hip.stream() for _ in range(2)]
    layers = [Layer(WeightFormat.F16, LENS, 48, seed=i, **FORMS[f]) for i, f in enumerate(("prefix", "window"))]
    want = []
    for e in layers:
        e.load(*STEPS[2])
        e.enqueue()
        want.append(e.check())
    for _ in range(5):
        for _ in range(4):
            for e, s in zip(layers, streams):
                e.enqueue(s.value)
        for e, s, w in zip(layers, streams, want):
            hip.call("hipStreamSynchronize", s)
            assert np.array_equal(e.get("out", np.float32, H), w)
    for s in streams:
        hip.call("hipStreamDestroy", s)
