"""GPU tests of the operators on paged K/V caches against float64 definitions (paged_ref.py): lengths from
nothing to several pages, head groups, page sizes, strides, both formats and types; slots that hold
no numbers, pages outside the pool, rows of no sequence."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as ref  # noqa: E402
from instantcua_amd import engine as eng  # noqa: E402
from instantcua_amd import paged  # noqa: E402
from instantcua_amd.modelfile import WeightFormat  # noqa: E402

pytestmark = pytest.mark.gpu
D = 128
NP = {paged.F32: np.float32, paged.F16: np.float16}
FMTS = [WeightFormat.F16, WeightFormat.Q8]
TYPES = [paged.F32, paged.F16]
dev = eng.DeviceBuffer.from_array


def upload(pool):
    return paged.PagedCache(pool.fmt, pool.n_kv, pool.page, pool.n_pages, dev(pool.data[0]), dev(pool.data[1]),
                            *([dev(s) for s in pool.scales] if pool.q8 else []))


def download(cache, pool):
    """The device pool's contents, as a host pool."""
    out = ref.Pool(pool.fmt, pool.n_kv, pool.page, pool.n_pages)
    out.data = [b.to_array(d.dtype, d.shape) for b, d in zip((cache.k, cache.v), pool.data)]
    if pool.q8:
        out.scales = [b.to_array(d.dtype, d.shape) for b, d in zip((cache.k_scales, cache.v_scales), pool.scales)]
    return out


def tables_of(kv_lens, page, rng, spare=2):
    """(table [n_seqs][width], pages of the pool): every sequence its own pages, in random order."""
    need = [-(-n // page) for n in kv_lens]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    width = max(1, max(need))
    table, at = np.zeros((len(need), width), np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, len(order)


# ---------------------------------------------------------------------------------------------
# store and load

STORE = [
    # heads, n_kv, page, tokens, rot, interleaved, norm
    (16, 8, 64, 8, 128, False, True),
    (16, 8, 16, 1, 128, False, True),
    (16, 8, 48, 77, 128, True, True),
    (12, 4, 32, 19, 64, False, True),
    (10, 2, 16, 5, 96, True, False),
    (5, 5, 16, 33, 8, False, True),
    (16, 1, 128, 3, 0, False, True),
    (0, 8, 64, 21, 128, False, True),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("types", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("case", STORE)
def test_store(fmt, types, case):
    heads, n_kv, page, T, rot, interleaved, norm = case
    rng = np.random.default_rng(hash(case) & 0xFFFF)
    type_, q_type = types
    pool = ref.Pool(fmt, n_kv, page, -(-T // page) + 3)
    cache = upload(pool)
    slots = rng.permutation(pool.n_pages * page)[:T].astype(np.int32)
    n = heads + 2 * n_kv
    stride, q_stride = n * D + 24, heads * D + 8  # rows with a gap behind them
    qkv = np.full((T, stride), np.nan, NP[type_])
    x = (rng.standard_normal((T, n, D)) * 2).astype(NP[type_])
    qkv[:, :n * D] = x.reshape(T, -1)
    w = [(1 + 0.3 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
    rows = 40
    pos, rope = rng.integers(0, rows, T).astype(np.int32), ref.rope_table(rows, rot)
    q = dev(np.full((T, q_stride), 7, NP[q_type]))
    cache.store(dev(qkv), T, dev(slots), n_heads=heads, q=q, q_norm=dev(w[0]) if norm else None,
                k_norm=dev(w[1]) if norm else None, rope=dev(rope) if rot else None, rope_rows=rows, pos=dev(pos),
                rot_dim=rot, interleaved=interleaved, type=type_, q_type=q_type, qkv_stride=stride, q_stride=q_stride)
    got_q = q.to_array(NP[q_type], (T, q_stride))
    assert (got_q[:, heads * D:] == 7).all()
    # fp32 arithmetic: a sum of 128 squares (2^-17 at most) and a few roundings, of the row's largest value.
    cs = rope[pos]
    want_q = ref.norm_rotate(x[:, :heads], w[0] if norm else None, cs, rot, interleaved)
    want = [ref.norm_rotate(x[:, heads:heads + n_kv], w[1] if norm else None, cs, rot, interleaved),
            x[:, heads + n_kv:].astype(np.float64)]
    fp32 = 2.0 ** -16
    got = got_q[:, :heads * D].reshape(T, heads, D).astype(np.float64)
    top = np.abs(want_q).max(-1, keepdims=True)
    assert (np.abs(got - want_q) <= fp32 * top + (2.0 ** -11 * np.abs(want_q) + 2.0 ** -25 if q_type else 0)).all()
    after = download(cache, pool)
    for i in range(2):
        y, top = after.values(i, slots), np.abs(want[i]).max(-1, keepdims=True)
        if fmt == WeightFormat.F16:
            assert (np.abs(y - want[i]) <= fp32 * top + 2.0 ** -11 * np.abs(want[i]) + 2.0 ** -25).all()
        else:  # half a step of a scale that is at most one fp16 step above amax / 127
            amax = np.abs(want[i]).reshape(T, n_kv, 4, 32).max(-1)
            step = np.repeat(after.scales[i][after.where(slots)].astype(np.float64), 32, axis=-1)
            assert (np.abs(y - want[i]) <= step / 2 * (1 + 2.0 ** -20) + fp32 * top).all()
            sc = after.scales[i][after.where(slots)].astype(np.float64)
            assert (sc >= amax / 127 * (1 - 2.0 ** -15)).all() and (sc <= amax / 127 * (1 + 2.0 ** -9)).all()
    # Nothing else was written.
    left = np.ones(pool.n_pages * page, bool)
    left[slots] = False
    w_ = after.where(np.nonzero(left)[0])
    for i in range(2):
        assert np.array_equal(after.data[i][w_], pool.data[i][w_], equal_nan=not pool.q8)
        assert np.isnan(after.scales[i][w_]).all()


def test_store_q8_has_the_bytes_of_the_quantiser():
    """Rows written as they are equal icua_quantize of the same fp32 matrix, byte for byte."""
    rng = np.random.default_rng(5)
    T, n_kv, page = 37, 8, 16
    x = (rng.standard_normal((T, 2 * n_kv, D)) * 10.0 ** rng.uniform(-6, 3, (T, 2 * n_kv, 1))).astype(np.float32)
    x[3] = 0
    x[4, 0, :32] = 127 * 0.25  # codes at the half steps' neighbours
    x[4, 0, 1:32] = (np.arange(31) + 0.5) * 0.25
    pool = ref.Pool(WeightFormat.Q8, n_kv, page, 3)
    cache = upload(pool)
    slots = rng.permutation(3 * page)[:T].astype(np.int32)
    cache.store(dev(x), T, dev(slots))
    after = download(cache, pool)
    codes, scales = eng.DeviceBuffer(x.size), eng.DeviceBuffer(x.size // 16)
    eng._check(eng.lib().icua_quantize(WeightFormat.Q8, dev(x).ptr, T * 2 * n_kv, D, codes.ptr, scales.ptr))
    codes = codes.to_array(np.int8, x.shape)
    scales = scales.to_array(np.uint16, x.shape[:2] + (4,))
    for i in range(2):
        half = slice(i * n_kv, (i + 1) * n_kv)
        assert np.array_equal(after.data[i][after.where(slots)], codes[:, half])
        assert np.array_equal(after.scales[i][after.where(slots)].view(np.uint16), scales[:, half])


@pytest.mark.parametrize("fmt", FMTS)
def test_store_leaves_out_tokens_without_a_slot_or_a_position(fmt):
    rng = np.random.default_rng(1)
    pool = ref.Pool(fmt, 2, 16, 2)
    cache = upload(pool)
    x = rng.standard_normal((6, 8, D)).astype(np.float32)
    slots = np.array([3, -1, 32, 2 ** 31 - 1, 5, 6], np.int32)  # the pool has 32 slots
    pos = np.array([0, 1, 2, 3, 4, -1], np.int32)               # and the table 4 rows
    q, rope = dev(np.zeros((6, 4, D), np.float32)), ref.rope_table(4, D)
    cache.store(dev(x), 6, dev(slots), n_heads=4, q=q, rope=dev(rope), rope_rows=4, pos=dev(pos))
    got = q.to_array(np.float32, (6, 4, D))
    want = ref.norm_rotate(x[:4, :4], None, rope[pos[:4]], D, False)
    assert (np.abs(got[:4] - want) <= 2.0 ** -16 * np.abs(want).max()).all()
    assert np.isnan(got[4:]).all()
    after = download(cache, pool)
    written = ~np.isnan(after.scales[0][..., 0] if pool.q8 else after.data[0][..., 0])
    assert written.sum() == 2 and written[0, :, 3].all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_kv,page,rows", [(8, 64, 1), (8, 16, 61), (3, 48, 130), (1, 16, 17)])
def test_load(fmt, type_, n_kv, page, rows):
    rng = np.random.default_rng(rows)
    pool = ref.Pool(fmt, n_kv, page, -(-rows // page) + 1)
    pool.fill(np.arange(pool.n_pages * page), rng)
    cache = upload(pool)
    slots = rng.permutation(pool.n_pages * page)[:rows].astype(np.int32)
    total = pool.n_pages * page
    given = slots.copy()
    if rows > 3:
        given[1], given[2] = -1, total  # neither is a slot: those rows stay as they are
    want = [pool.values(i, slots) for i in range(2)]
    for heads_first in (False, True):
        shape = (n_kv, rows + 1, D) if heads_first else (rows, n_kv, D)
        k, v = (dev(np.full(shape, 3, NP[type_])) for _ in range(2))
        strides = dict(token_stride=D, head_stride=(rows + 1) * D) if heads_first else {}
        cache.load(dev(given), rows, k, v, type=type_, **strides)
        cache.load(dev(given), rows, None, v, type=type_, **strides)  # one of them alone
        for b, w in zip((k, v), want):
            got = b.to_array(NP[type_], shape)
            if heads_first:
                assert (got[:, rows] == 3).all()
                got = got[:, :rows].transpose(1, 0, 2)
            w = w.astype(np.float32).astype(NP[type_])  # s q is exact in fp32, then one rounding
            if rows > 3:
                assert (got[1:3] == 3).all()
                got, w = np.delete(got, (1, 2), 0), np.delete(w, (1, 2), 0)
            assert np.array_equal(got, w)


# ---------------------------------------------------------------------------------------------
# attention

ATTENTION = [
    # heads, n_kv, page, [(new tokens, slots)]
    (16, 8, 64, [(1, 1)]),
    (16, 8, 64, [(1, 300), (1, 17), (1, 64), (1, 1), (1, 2)]),
    (16, 8, 16, [(1, 2000), (0, 50), (1, 0), (1, 129)]),
    (16, 8, 64, [(8, 700), (3, 3), (5, 100)]),
    (16, 8, 48, [(9, 9), (1, 250), (41, 300)]),
    (4, 4, 32, [(20, 100), (16, 16), (17, 40)]),
    (12, 4, 16, [(6, 90), (1, 31), (30, 33)]),
    (10, 2, 128, [(3, 500), (4, 4)]),
    (16, 1, 16, [(1, 400), (1, 3)]),
    (16, 1, 16, [(7, 200)]),
    (6, 2, 32, [(5, 2), (3, 0), (2, 40)]),  # more new tokens than slots: the first rows see nothing
    (2, 2, 16, [(150, 333), (1, 40)]),
    (16, 8, 64, [(130, 200)]),
]


def run_attention(pool, q, q_lens, kv_lens, table, type_, extra=0, cache=None, stream=0, **kw):
    """The operator's outputs, from a buffer with `extra` rows behind the last sequence's (kept at 7)."""
    heads, T = q.shape[1], int(np.sum(q_lens))
    cache = cache or upload(pool)
    stride = heads * D + 16
    qb = np.full((T + extra, stride), np.nan, NP[type_])
    qb[:T, :heads * D] = q.reshape(T, -1)
    out = dev(np.full((T + extra, stride), 7, NP[type_]))
    start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    sizes = dict(max_q=int(max(q_lens)), max_kv=max(1, int(max(kv_lens))))
    n = cache.attention_work(heads, len(q_lens), T + extra, table_width=table.shape[1], **sizes)
    work = dev(np.full(n + 64, 0xFF, np.uint8)) if n else None
    cache.attention(dev(qb), out, heads, dev(start), dev(np.asarray(kv_lens, np.int32)), dev(table), len(q_lens),
                    T + extra, table.shape[1], type=type_, q_stride=stride, out_stride=stride, work=work,
                    stream=stream, **sizes, **kw)
    got = out.to_array(NP[type_], (T + extra, stride))
    assert (got[T:] == 7).all() and (got[:, heads * D:] == 7).all()
    if n:
        assert (work.to_array(np.uint8, (n + 64,))[n:] == 0xFF).all()
    return got[:T, :heads * D].reshape(T, heads, D).astype(np.float64)


def filled(fmt, n_kv, page, kv_lens, rng):
    table, pages = tables_of(kv_lens, page, rng)
    pool = ref.Pool(fmt, n_kv, page, pages)
    for row, n in zip(table, kv_lens):
        p = np.arange(n)
        pool.fill(row[p // page].astype(np.int64) * page + p % page, rng)
    return pool, table


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(fmt, type_, case):
    """Every slot that no sequence uses holds NaN, the rest of the last page too."""
    heads, n_kv, page, lens = ATTENTION[case]
    rng = np.random.default_rng(100 + case)
    q_lens, kv_lens = zip(*lens)
    pool, table = filled(fmt, n_kv, page, kv_lens, rng)
    q = (rng.standard_normal((sum(q_lens), heads, D)) * 1.5).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, extra=case % 3)
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table)
    tol = ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)
    assert np.isfinite(got).all() and np.abs(got - want).max() <= tol


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("scale,size", [(0.5, 4.0), (1e-3, 1.0), (-0.1, 1.0), (1e4, 1e-4), (2e-37, 1e37)])
def test_attention_scales(fmt, type_, scale, size):
    """Steep and flat softmaxes; queries far from 1 in size (fp32 ones beyond fp16's range)."""
    if type_ == paged.F16 and size > 1e4:
        size, scale = 8e3, 1e-5
    rng = np.random.default_rng(9)
    q_lens, kv_lens = (1, 4, 20), (333, 40, 100)
    pool, table = filled(fmt, 4, 16, kv_lens, rng)
    q = (rng.standard_normal((25, 8, D)) * size).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, scale=scale)
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table, scale=scale)
    assert np.abs(got - want).max() <= ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("m", [6, 40])
def test_attention_of_tokens_before_one_that_is_no_number(fmt, type_, what, m):
    """A new token whose key and value are no numbers spoils its own outputs and those of later tokens
    of its sequence, no others."""
    rng = np.random.default_rng(3)
    q_lens, kv_lens = (m, 2), (100, 30)
    pool, table = filled(fmt, 2, 16, kv_lens, rng)
    q = rng.standard_normal((m + 2, 4, D)).astype(NP[type_])
    bad = 4  # token 4 of the first sequence
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table)
    slot = 100 - m + bad
    at = table[0, slot // 16], slice(None), slot % 16
    for i in range(2):
        if pool.q8:
            pool.scales[i][at] = what
        else:
            pool.data[i][at] = what
    got = run_attention(pool, q, q_lens, kv_lens, table, type_)
    tol = ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)
    fine = [i for i in range(m + 2) if i < bad or i >= m]
    assert np.abs(got[fine] - want[fine]).max() <= tol
    if np.isnan(what):
        assert np.isnan(got[bad:m]).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 30])
def test_attention_leaves_out_pages_outside_the_pool(fmt, m):
    rng = np.random.default_rng(4)
    q_lens, kv_lens = (m, m, 1), (200, 100, 64)
    pool, table = filled(fmt, 2, 32, kv_lens, rng)
    table[0, 1], table[0, 4], table[1, 0] = -1, pool.n_pages, 2 ** 31 - 1
    table[2, :2] = -5  # nothing is left of this one
    q = rng.standard_normal((2 * m + 1, 4, D)).astype(np.float32)
    got = run_attention(pool, q, q_lens, kv_lens, table, paged.F32)
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table)
    assert (got[2 * m] == 0).all()
    assert np.abs(got - want).max() <= ref.attention_tol(False, pool.q8, reach, vmax)


def test_attention_with_lengths_and_starts_outside_the_buffers():
    """Lengths past max_kv and starts past n_tokens are cut: nothing outside the buffers is read or
    written, the other sequences are right."""
    rng = np.random.default_rng(6)
    pool, table = filled(WeightFormat.F16, 2, 16, (64, 64), rng)
    q = rng.standard_normal((3, 4, D)).astype(np.float32)
    cache = upload(pool)
    out = dev(np.full((3, 4, D), 7, np.float32))
    sizes = dict(max_q=1, max_kv=64)
    work = eng.DeviceBuffer(max(16, cache.attention_work(4, 3, 3, table_width=4, **sizes)))
    start, kv = np.array([0, 1, 2, 9], np.int32), np.array([64, 5000, -7], np.int32)
    full = np.concatenate([table, table[:1]])
    cache.attention(dev(q), out, 4, dev(start), dev(kv), dev(full), 3, 3, 4, work=work, **sizes)
    got = out.to_array(np.float32, (3, 4, D)).astype(np.float64)
    want, reach, vmax = ref.attention(pool, q, (1, 1, 1), (64, 64, 0), full)
    assert np.abs(got - want).max() <= ref.attention_tol(False, False, reach, vmax)


def test_sequences_may_share_pages():
    """Two sequences with a common prefix: their outputs are those of sequences with pages of their own."""
    rng = np.random.default_rng(8)
    pool, table = filled(WeightFormat.F16, 2, 32, (96, 40), rng)
    shared = np.array([[table[0, 0], table[0, 1], table[0, 2]], [table[0, 0], table[1, 0], table[1, 1]]], np.int32)
    q = rng.standard_normal((2, 4, D)).astype(np.float32)
    got = run_attention(pool, q, (1, 1), (96, 72), shared, paged.F32)
    want, reach, vmax = ref.attention(pool, q, (1, 1), (96, 72), shared)
    assert np.abs(got - want).max() <= ref.attention_tol(False, False, reach, vmax)


def test_attention_repeats_to_the_bit():
    rng = np.random.default_rng(12)
    q_lens, kv_lens = (1, 1, 40), (1500, 700, 900)
    pool, table = filled(WeightFormat.Q8, 8, 64, kv_lens, rng)
    q = rng.standard_normal((42, 16, D)).astype(np.float32)
    cache = upload(pool)
    first = run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=cache)
    for _ in range(3):
        assert np.array_equal(run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=cache), first)
