"""GPU tests of the operators on paged K/V caches together, as a server uses them: sessions that grow by chunks
and single tokens, captured graphs replayed with new contents, streams side by side; and batches and caches
beyond what one wave, one workgroup or 32 bits of a byte offset cover.  Definitions in paged_ref.py."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as ref  # noqa: E402
from instantcua_amd import engine as eng  # noqa: E402
from instantcua_amd import paged, synth  # noqa: E402
from instantcua_amd.modelfile import Dims, TensorID, WeightFormat  # noqa: E402
from test_gpu_paged import D, FMTS, NP, TYPES, dev, download, filled, run_attention, tables_of, upload  # noqa: E402

pytestmark = pytest.mark.gpu


def put(buffer, a):
    """New contents of a device buffer."""
    a = np.ascontiguousarray(a)
    assert a.nbytes <= buffer.nbytes
    eng._check(eng.lib().icua_memcpy_h2d(buffer.ptr, a.ctypes.data, a.nbytes))


class Hip:
    """Streams and graphs of the HIP runtime that the library runs on."""

    def __init__(self):
        eng.lib()
        with open("/proc/self/maps") as f:
            self.so = C.CDLL(next(x.split()[-1] for x in f if "libamdhip64" in x))

    def call(self, name, *args):
        assert getattr(self.so, name)(*args) == 0, name

    def stream(self):
        s = C.c_void_p()
        self.call("hipStreamCreate", C.byref(s))
        return s

    def capture(self, stream, enqueue):
        graph, ready = C.c_void_p(), C.c_void_p()
        self.call("hipStreamBeginCapture", stream, 1)
        enqueue(stream.value)
        self.call("hipStreamEndCapture", stream, C.byref(graph))
        self.call("hipGraphInstantiate", C.byref(ready), graph, None, None, C.c_size_t(0))
        self.call("hipGraphDestroy", graph)
        return ready


class Sessions:
    """A pool with room for `lens` slots a session, and one call's buffers for up to `tokens` new tokens, at
    fixed addresses."""

    def __init__(self, fmt, type_, heads, n_kv, page, lens, tokens, rng, seed=1):
        self.type, self.heads, self.n_kv, self.lens, self.tokens = type_, heads, n_kv, lens, tokens
        self.table, pages = tables_of(lens, page, np.random.default_rng(seed))
        self.pool = ref.Pool(fmt, n_kv, page, pages)
        self.cache = upload(self.pool)
        self.rope_rows = max(lens)
        self.rope = dev(ref.rope_table(self.rope_rows, D))
        self.norms = [dev((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2)]
        n = heads + 2 * n_kv
        self.qkv, self.q = (eng.DeviceBuffer(tokens * k * D * 4) for k in (n, heads))
        self.out = dev(np.full((tokens, heads, D), 7, NP[type_]))
        self.pos, self.slots = (eng.DeviceBuffer(tokens * 4) for _ in range(2))
        self.start, self.kv = eng.DeviceBuffer((len(lens) + 1) * 4), eng.DeviceBuffer(len(lens) * 4)
        self.tables = dev(self.table)
        self.sizes = dict(max_q=tokens, max_kv=max(lens))
        self.work = eng.DeviceBuffer(max(16, cache_work(self.cache, heads, len(lens), tokens, self.table.shape[1], self.sizes)))
        self.have = [0] * len(lens)

    def load(self, x, news):
        """The next `news` tokens of every session are x [sum(news)][heads + 2 n_kv][128]; tokens behind them
        have no slot."""
        T = sum(news)
        put(self.qkv, x.astype(NP[self.type]))
        pos, slots = np.zeros(self.tokens, np.int32), np.full(self.tokens, -1, np.int32)
        pos[:T] = np.concatenate([np.arange(h, h + n) for h, n in zip(self.have, news)])
        slots[:T] = np.concatenate([self.cache.slots(t, h, n) for t, h, n in zip(self.table, self.have, news)])
        self.have = [h + n for h, n in zip(self.have, news)]
        for b, a in ((self.pos, pos), (self.slots, slots), (self.kv, np.array(self.have, np.int32)),
                     (self.start, np.concatenate([[0], np.cumsum(news)]).astype(np.int32))):
            put(b, a)

    def enqueue(self, stream=0):
        c = self.cache
        c.store(self.qkv, self.tokens, self.slots, n_heads=self.heads, q=self.q, q_norm=self.norms[0], k_norm=self.norms[1],
                rope=self.rope, rope_rows=self.rope_rows, pos=self.pos, type=self.type, q_type=self.type, stream=stream)
        c.attention(self.q, self.out, self.heads, self.start, self.kv, self.tables, len(self.lens), self.tokens,
                    self.table.shape[1], type=self.type, work=self.work, stream=stream, **self.sizes)

    def result(self):
        return self.out.to_array(NP[self.type], (self.tokens, self.heads, D))

    def queries(self):
        return self.q.to_array(NP[self.type], (self.tokens, self.heads, D))


def cache_work(cache, heads, n_seqs, tokens, width, sizes):
    return cache.attention_work(heads, n_seqs, tokens, table_width=width, **sizes)


STEPS = [(37, 5, 64), (1, 1, 20), (1, 1, 1), (4, 1, 1), (0, 30, 1), (1, 1, 1)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
def test_sessions_grow_by_chunks_and_tokens(fmt, type_):
    """Every step's outputs are the definition's over what the cache then holds; at the end one pass over all
    of a session's queries gives what the steps gave."""
    rng = np.random.default_rng(21)
    lens = [sum(s[i] for s in STEPS) for i in range(3)]
    run = Sessions(fmt, type_, 8, 4, 16, lens, 110, rng)
    past_q, past_out = [[] for _ in lens], [[] for _ in lens]
    for news in STEPS:
        T = sum(news)
        run.load(rng.standard_normal((T, 16, D)), news)
        before = run.result()
        run.enqueue()
        got, q = run.result(), run.queries()[:T]
        assert np.array_equal(got[T:], before[T:])  # rows of no sequence
        pool = download(run.cache, run.pool)
        want, reach, vmax = ref.attention(pool, q, news, run.have, run.table)
        tol = ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)
        assert np.abs(got[:T] - want).max() <= tol
        at = 0
        for i, n in enumerate(news):
            past_q[i].append(q[at:at + n])
            past_out[i].append(got[at:at + n])
            at += n
    q = np.concatenate([x for s in past_q for x in s])
    steps = np.concatenate([x for s in past_out for x in s]).astype(np.float64)
    whole = run_attention(pool, q, lens, lens, run.table, type_, cache=run.cache)
    want, reach, vmax = ref.attention(pool, q, lens, lens, run.table)
    tol = ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)
    assert np.abs(whole - want).max() <= tol and np.abs(whole - steps).max() <= 2 * tol


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("tokens", [3, 40])  # of few rows alone, and a padded batch
def test_a_captured_step_replays_with_new_contents(fmt, tokens):
    """Store and attention in one graph, replayed over three sessions that grow; between the replays the same
    step runs eagerly on a second pool, and gives the same to the bit."""
    hip, rng = Hip(), np.random.default_rng(22)
    lens = (700, 90, 41)
    a, b = (Sessions(fmt, paged.F32, 8, 4, 16, lens, tokens, np.random.default_rng(2)) for _ in range(2))
    stream = hip.stream()
    graph = hip.capture(stream, a.enqueue)
    assert (a.result() == 7).all()  # nothing ran yet
    start = (600, 50, 0)
    for s in (a, b):
        s.have = list(start)
    first = np.random.default_rng(3)
    for s in (a, b):  # what the sessions hold before
        for t, n in zip(s.table, start):
            p = np.arange(n)
            s.pool.fill(t[p // 16].astype(np.int64) * 16 + p % 16, first if s is a else np.random.default_rng(3))
    b.pool.data, b.pool.scales = [d.copy() for d in a.pool.data], [d.copy() for d in a.pool.scales]
    for s in (a, b):
        put(s.cache.k, s.pool.data[0]), put(s.cache.v, s.pool.data[1])
        if s.pool.q8:
            put(s.cache.k_scales, s.pool.scales[0]), put(s.cache.v_scales, s.pool.scales[1])
    for step in range(4):
        news = [(1, 1, 1), (0, 1, 1), (1, 1, 1), (1, 0, 1)][step] if tokens == 3 else [(9, 1, 8), (1, 1, 30), (1, 1, 1), (20, 12, 1)][step]
        x = rng.standard_normal((sum(news), 16, D))
        a.load(x, news), b.load(x, news)
        hip.call("hipGraphLaunch", graph, stream)
        b.enqueue()
        hip.call("hipStreamSynchronize", stream)
        got, want = a.result()[:sum(news)], b.result()[:sum(news)]
        assert np.array_equal(got, want)
        pool = download(a.cache, a.pool)
        exact, reach, vmax = ref.attention(pool, a.queries()[:sum(news)], news, a.have, a.table)
        assert np.abs(got - exact).max() <= ref.attention_tol(False, pool.q8, reach, vmax)
    hip.call("hipGraphExecDestroy", graph)
    hip.call("hipStreamDestroy", stream)


def test_streams_side_by_side():
    """Calls on two streams over one pool, each with its own workspace, give what each gives alone."""
    hip, rng = Hip(), np.random.default_rng(23)
    q_lens, kv_lens = (1, 1, 1, 1), (3000, 1500, 2000, 64)
    pool, table = filled(WeightFormat.F16, 4, 64, kv_lens, rng)
    cache, streams = upload(pool), [hip.stream(), hip.stream()]
    sizes = dict(max_q=1, max_kv=3000)
    n = cache.attention_work(8, 4, 4, table_width=table.shape[1], **sizes)
    start, kv, tables = dev(np.arange(5, dtype=np.int32)), dev(np.array(kv_lens, np.int32)), dev(table)
    qs = [rng.standard_normal((4, 8, D)).astype(np.float32) for _ in range(2)]
    alone = [run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=cache) for q in qs]
    bufs = [(dev(q), eng.DeviceBuffer(q.nbytes), eng.DeviceBuffer(n)) for q in qs]
    for _ in range(5):
        for (q, out, work), s in zip(bufs, streams):
            for _ in range(3):
                cache.attention(q, out, 8, start, kv, tables, 4, 4, table.shape[1], work=work, stream=s.value, **sizes)
        for s in streams:
            hip.call("hipStreamSynchronize", s)
        for (_, out, _), want in zip(bufs, alone):
            assert np.array_equal(out.to_array(np.float32, (4, 8, D)), want)
    for s in streams:
        hip.call("hipStreamDestroy", s)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_kv,max_new", [(1, 1), (16, 1), (16, 3), (2, 40)])
def test_attention_of_many_sequences(fmt, type_, n_kv, max_new):
    """More sequences than a wave has lanes, of mixed lengths, some with no new token or no slot: workgroups
    with several sequences, sequences with several workgroups, both kinds of sequences in one batch."""
    rng = np.random.default_rng(n_kv + max_new)
    n = 141
    kv_lens = [int(x) for x in np.exp(rng.uniform(0, np.log(700), n))]
    kv_lens[5], kv_lens[64], kv_lens[100] = 0, 1900, 1
    q_lens = [int(x) for x in rng.integers(0, 2, n)] if max_new == 1 else [int(x) for x in rng.integers(0, max_new + 1, n)]
    q_lens = [min(m, max(1, k)) for m, k in zip(q_lens, kv_lens)]
    q_lens[5] = q_lens[64] = q_lens[140] = 1
    pool, table = filled(fmt, n_kv, 16, kv_lens, rng)
    q = rng.standard_normal((sum(q_lens), 2 * n_kv if n_kv < 16 else n_kv, D)).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, extra=3)
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table)
    assert np.abs(got - want).max() <= ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m", [1, 9])
def test_attention_of_a_long_sequence(fmt, type_, m):
    """One sequence over more units than there are partials: every workgroup has several."""
    rng = np.random.default_rng(31)
    kv = 41003
    pool, table = filled(fmt, 1, 64, (kv,), rng)
    q = rng.standard_normal((m, 2, D)).astype(NP[type_])
    got = run_attention(pool, q, (m,), (kv,), table, type_)
    want, reach, vmax = ref.attention(pool, q, (m,), (kv,), table)
    assert np.abs(got - want).max() <= ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m", [1, 70])
@pytest.mark.parametrize("low,high", [(1e-4, 1e-3), (0.5, 300.0), (1e-5, 100.0)])
def test_attention_over_q8_values_of_any_size(type_, m, low, high):
    """Scales of V far below and above 1, spread over the groups and slots: what the groups of small values
    give is held to their own size."""
    rng = np.random.default_rng(32)
    q_lens, kv_lens = (m, 2), (300, 64)
    pool, table = filled(WeightFormat.Q8, 2, 32, kv_lens, rng)
    sc = np.exp(rng.uniform(np.log(low), np.log(high), pool.scales[1].shape))
    if low < 1e-4:  # groups of a size each
        sc = np.broadcast_to(np.array([low, 1e-2, 1.0, high]) * 1.0, pool.scales[1].shape) * rng.uniform(0.5, 1, pool.scales[1].shape)
    pool.scales[1] = np.where(np.isnan(pool.scales[1]), np.float16(np.nan), sc.astype(np.float16))
    q = rng.standard_normal((m + 2, 4, D)).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_)
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table)
    if low >= 1e-4:
        assert np.abs(got - want).max() <= ref.attention_tol(type_ == paged.F16, True, reach, vmax)
        return
    tol = ref.attention_tol(type_ == paged.F16, True, reach, 1.0)
    for g in range(4):
        dims = slice(32 * g, 32 * g + 32)
        top = 127 * float(np.nanmax(pool.scales[1][..., g].astype(np.float64)))
        # fp16 outputs below 2^-14 step by 2^-24.  A maximum that stands 2^7 above (the power of two of 100)
        # leaves the largest products of probability and scale at 2^(9 - 7) low = 2^2 1e-5 = 2^-15: fp16 steps of
        # 2^-24 there, half a step 2^-25, is 2^-10 of it.
        small = 2.0 ** -25 + 2.0 ** -10 * top if type_ == paged.F16 and g == 0 else 0.0
        assert np.abs(got - want)[..., dims].max() <= tol * top + small


def test_a_pool_of_more_than_2_to_the_31_bytes():
    """Pages at the far end of K and V of 2.3 GB each."""
    rng = np.random.default_rng(33)
    n_kv, page, pages = 8, 64, 18000
    assert n_kv * page * pages * D * 2 > 2 ** 31
    cache = paged.PagedCache(WeightFormat.F16, n_kv, page, pages)
    table = np.array([[pages - 1, 0, pages - 2], [17000, 16999, 3]], np.int32)
    kv_lens, T = (150, 130), 280
    x = rng.standard_normal((T, 2 * n_kv, D)).astype(np.float32)
    slots = np.concatenate([cache.slots(t, 0, n) for t, n in zip(table, kv_lens)])
    cache.store(dev(x), T, dev(slots))
    k, v = (eng.DeviceBuffer(T * n_kv * D * 4) for _ in range(2))
    cache.load(dev(slots), T, k, v)
    got = [b.to_array(np.float32, (T, n_kv, D)) for b in (k, v)]
    assert np.array_equal(got[0], x[:, :n_kv].astype(np.float16)) and np.array_equal(got[1], x[:, n_kv:].astype(np.float16))
    pool = ref.Pool(WeightFormat.F16, n_kv, page, 6)  # the six pages, as pages 0 .. 5 of a small pool
    small = np.arange(6, dtype=np.int32).reshape(2, 3)
    at = 0
    for t, n in zip(small, kv_lens):
        p = np.arange(n)
        w = pool.where(t[p // page].astype(np.int64) * page + p % page)
        for i in range(2):
            pool.data[i][w] = got[i][at:at + n]
        at += n
    for q_lens in ((1, 1), (40, 1)):
        q = rng.standard_normal((sum(q_lens), 16, D)).astype(np.float32)
        out = run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=cache)
        want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, small)
        assert np.abs(out - want).max() <= ref.attention_tol(False, False, reach, vmax)
    cache.k.free(), cache.v.free()


@pytest.mark.parametrize("fmt", FMTS)
def test_one_page_may_hold_a_whole_session(fmt):
    """A pool of one page of all slots, as the engine's contiguous cache lays out a layer."""
    rng = np.random.default_rng(34)
    pool, table = filled(fmt, 8, 1024, (777,), rng)
    q = rng.standard_normal((1, 16, D)).astype(np.float32)
    got = run_attention(pool, q, (1,), (777,), table, paged.F32)
    want, reach, vmax = ref.attention(pool, q, (1,), (777,), table)
    assert np.abs(got - want).max() <= ref.attention_tol(False, pool.q8, reach, vmax)


@pytest.mark.parametrize("pos,n", [(29, 3), (700, 1), (1000, 8)])
def test_the_operators_compute_the_engines_layer(pos, n):
    """The engine's fused q|k|v rows of a layer pass, through store and attention on a pool of one page that holds
    its cache: the engine's K/V rows and attention output.

    Values are rounded from the same fp32 on both sides.  Keys go through the norm's sum and the table's angles
    first, which differ in their last bits, so some lie on the other side of a rounding: one fp16 step, in at
    most 2 % of them, and the attention over them within 1e-4 of its largest magnitude, as the engine's own
    stages are held to their oracle."""
    img = synth.build_model_image(WeightFormat.Q4, n_layers=2, tag="q4-small")
    ctx, layer = 1024, 1
    kc, vc = (synth.fp16_normal((8, pos, D), f"pu-{k}", pos) for k in "kv")
    x = synth.fp16_normal((n, Dims.hidden), "pu-x", n).astype(np.float32)
    with eng.Engine(flags=0, image=img, max_context=ctx) as e:
        e.write_kv(layer, 0, 0, kc)
        e.write_kv(layer, 1, 0, vc)
        e.layer_step(layer, x, pos)
        qkv, want = e.read_buffer("qkv")[:n], e.read_buffer("attn")[:n].reshape(n, 16, D)
        rows = [e.read_kv(layer, kind, pos, n) for kind in range(2)]
    pool = ref.Pool(WeightFormat.F16, 8, ctx, 1)
    pool.data[0][0, :, :pos], pool.data[1][0, :, :pos] = kc, vc
    cache = upload(pool)
    norms = [dev(synth.tensor_view(img, TensorID.llm_layer(layer, i)).view(np.float32).copy()) for i in (TensorID.q_norm, TensorID.k_norm)]
    # The engine's table: the angle is a product in fp32 (Engine.swift:121-125), up to 2^-14 off at slot 1000.
    angle = (np.arange(ctx, dtype=np.float32)[:, None] * (Dims.rope_theta ** -(np.arange(0, D, 2) / D)).astype(np.float32)).astype(np.float64)
    rope = np.stack([np.cos(angle), np.sin(angle)], axis=-1).astype(np.float32)
    at, q, out = np.arange(pos, pos + n, dtype=np.int32), eng.DeviceBuffer(n * 16 * D * 4), eng.DeviceBuffer(n * 16 * D * 4)
    cache.store(dev(qkv), n, dev(at), n_heads=16, q=q, q_norm=norms[0], k_norm=norms[1], rope=dev(rope), rope_rows=ctx, pos=dev(at))
    sizes = dict(max_q=n, max_kv=ctx)
    work = eng.DeviceBuffer(max(16, cache.attention_work(16, 1, n, table_width=1, **sizes)))
    cache.attention(q, out, 16, dev(np.array([0, n], np.int32)), dev(np.array([pos + n], np.int32)), dev(np.zeros((1, 1), np.int32)),
                    1, n, 1, work=work, **sizes)
    after = download(cache, pool)
    got_k, got_v = (after.data[i][0, :, pos:pos + n] for i in range(2))
    assert np.array_equal(got_v.view(np.uint16), rows[1].view(np.uint16))
    k, w = got_k.astype(np.float32), rows[0].astype(np.float32)
    step = np.spacing(np.abs(rows[0])).astype(np.float32)
    assert (np.abs(k - w) <= step + 1e-6 * np.abs(w).max()).all() and (k != w).mean() < 2e-2
    got = out.to_array(np.float32, (n, 16, D))
    assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [8, 33])
def test_fp32_probabilities_keep_both_parts(fmt, m):
    """Flat softmaxes over few slots, where a probability whose fp16 parts do not add up to it would show: the
    outputs are within the fp32 bound (2^-12 / 8 of a value, for a part rounded otherwise than the other
    expects among eight slots, is ten times as much), over enough rows for roundings next to a tie."""
    rng = np.random.default_rng(35)
    lens = (m,) * 60
    pool, table = filled(fmt, 4, 48, lens, rng)
    q = rng.standard_normal((60 * m, 8, D)).astype(np.float32)
    got = run_attention(pool, q, lens, lens, table, paged.F32, scale=1e-3)
    want, reach, vmax = ref.attention(pool, q, lens, lens, table, scale=1e-3)
    assert np.abs(got - want).max() <= ref.attention_tol(False, pool.q8, reach, vmax)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 20])
def test_attention_joins_any_number_of_partials(fmt, type_, m):
    """Sequences of 1 .. 64 units of 128 slots, each alone in a call, so that every number of partials is joined."""
    rng = np.random.default_rng(36)
    pool, table = filled(fmt, 1, 128, (64 * 128,), rng)
    q = rng.standard_normal((m, 2, D)).astype(NP[type_])
    cache = upload(pool)
    for units in (1, 2, 3, 16, 17, 31, 32, 33, 34, 35, 47, 48, 49, 62, 63, 64):
        kv = 128 * units - 5
        got = run_attention(pool, q, (m,), (kv,), table, type_, cache=cache)
        want, reach, vmax = ref.attention(pool, q, (m,), (kv,), table)
        assert np.abs(got - want).max() <= ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax), units


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("q_lens", [(1, 0, 1, 2), (1, 0, 60, 2)])
def test_bounds_may_be_loose(fmt, type_, q_lens):
    """A padded batch: sequences without tokens or slots behind the others, tables wider than any sequence with
    anything in the unused entries, no bound on tokens or slots given."""
    rng = np.random.default_rng(37)
    kv_lens = (900, 40, 333, 2)
    pool, table = filled(fmt, 2, 32, kv_lens, rng)
    wide = rng.integers(-2 ** 31, 2 ** 31 - 1, (7, 200)).astype(np.int32)
    for i, n in enumerate(kv_lens):
        wide[i, :-(-n // 32)] = table[i, :-(-n // 32)]
    T, room = sum(q_lens), sum(q_lens) + 30
    q = np.full((room, 4, D), np.nan, NP[type_])
    q[:T] = rng.standard_normal((T, 4, D))
    cache, out = upload(pool), dev(np.full((room, 4, D), 7, NP[type_]))
    start = np.concatenate([[0], np.cumsum(q_lens), [T] * 3]).astype(np.int32)
    n = cache.attention_work(4, 7, room, table_width=200)
    work = dev(np.full(n + 64, 0xFF, np.uint8))
    cache.attention(dev(q), out, 4, dev(start), dev(np.array(kv_lens + (0, 50, 0), np.int32)), dev(wide), 7, room, 200,
                    type=type_, work=work)
    got = out.to_array(NP[type_], (room, 4, D))
    assert (got[T:] == 7).all() and (work.to_array(np.uint8, (n + 64,))[n:] == 0xFF).all()
    want, reach, vmax = ref.attention(pool, q[:T], q_lens, kv_lens, table)
    assert np.abs(got[:T] - want).max() <= ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)
