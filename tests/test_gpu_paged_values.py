"""GPU tests of the operators on paged K/V caches where values or batches are unusual.  Definitions in paged_ref.py."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_bounds as bounds  # noqa: E402
import paged_ref as ref  # noqa: E402
from instantcua_amd import paged  # noqa: E402
from instantcua_amd.modelfile import WeightFormat  # noqa: E402
from test_gpu_paged import D, FMTS, NP, TYPES, dev, download, filled, run_attention, upload  # noqa: E402

pytestmark = pytest.mark.gpu


# New tokens, slots of the first sequence and the slots that are spoiled, one at a time: prompts whose tokens see
# the halves of 64 slots in part or in full, a follow-up that does, drafts and single tokens.
SPOILED = [
    (128, 128, (10, 63, 70, 127)),
    (300, 300, (10, 100, 140, 200, 299)),
    (41, 1248, (500, 1160, 1210, 1240)),
    (6, 100, (50, 96)),
    (1, 300, (7, 299)),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("case", range(len(SPOILED)))
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(fmt, type_, what, case):
    """V alone is spoiled (its key is an ordinary one): every token that sees the slot gives no number in those
    dims, every other token and dim what it gives without."""
    rng = np.random.default_rng(51)
    m, kv, slots = SPOILED[case]
    q_lens, kv_lens = (m, 3), (kv, 40)
    pool, table = filled(fmt, 2, 16, kv_lens, rng)
    q = rng.standard_normal((m + 3, 4, D)).astype(NP[type_])
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table)
    tol = ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)
    for slot in slots:
        at = table[0, slot // 16], 1, slot % 16
        if pool.q8:
            dims, kept = slice(64, 96), pool.scales[1][at].copy()
            pool.scales[1][at][2] = what
        else:
            dims, kept = slice(37, 38), pool.data[1][at].copy()
            pool.data[1][at][37] = what
        got = run_attention(pool, q, q_lens, kv_lens, table, type_)
        sees = np.zeros(got.shape, bool)
        sees[max(0, slot - (kv - m)):m, 2:, dims] = True  # KV head 1: query heads 2 and 3
        assert not np.isfinite(got[sees]).any(), slot
        assert np.abs(got - want)[~sees].max() <= tol, slot
        if pool.q8:
            pool.scales[1][at] = kept
        else:
            pool.data[1][at] = kept


def by_group(x):
    return x.reshape(*x.shape[:-1], 4, 32)


def of_sequences(pool, q, q_lens, kv_lens, table, got, floor=0.0, scale=None, type_=paged.F32):
    """Outputs of every sequence against the definition, groups of 32 dims by themselves."""
    group, at = q.shape[1] // pool.n_kv, 0
    for s, (m, n) in enumerate(zip(q_lens, kv_lens)):
        want, reach, _ = ref.attention(pool, q[at:at + m], (m,), (n,), table[s:s + 1], scale=scale)
        bound = bounds.rms_bound(type_ == paged.F16, pool.q8, bounds.chunked(m, group), reach, n)
        out = got[at:at + m].copy()
        if type_ == paged.F16:  # outputs that round to infinities; next to the border (2^-9 are two and more bounds) either may be
            assert (out == np.copysign(np.inf, want))[np.abs(want) > 65520 * (1 + 2.0 ** -9)].all()
            big = np.abs(want) > 65520 * (1 - 2.0 ** -9)
            out[big] = want[big] = 0
        bounds.check(by_group(out), by_group(want), bound, floor)
        at += m


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m", [1, 6])
@pytest.mark.parametrize("size", [516.0, -516.0, 3000.0, 65504.0])
def test_q8_values_beyond_fp16(type_, m, size):
    """Groups whose values (code times scale) are beyond what fp16 holds are exact for single tokens and drafts,
    also for tokens that do not see them."""
    q8_values_beyond_fp16(type_, m, size)


def q8_values_beyond_fp16(type_, m, size):
    rng = np.random.default_rng(52)
    q_lens, kv_lens = (m, 2), (300, 64)
    pool, table = filled(WeightFormat.Q8, 2, 32, kv_lens, rng)
    for slot, g in ((20, 1), (299 - m // 2, 2), (299, 0)):
        at = table[0, slot // 32], slice(None), slot % 32
        pool.scales[1][at][..., g] = size
        pool.data[1][at][..., 32 * g:32 * g + 32:5] = 127
        pool.data[1][at][..., 32 * g + 1:32 * g + 32:5] = -127
    q = (0.3 * rng.standard_normal((m + 2, 4, D))).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_)
    of_sequences(pool, q, q_lens, kv_lens, table, got, type_=type_)


def test_a_stored_value_of_65504_is_read_alike():
    """The largest value that the store takes, from a q8 pool: single tokens, drafts, chunks and an fp32 load
    have what code and scale say; an fp16 load rounds it."""
    rng = np.random.default_rng(53)
    T, page = 60, 16
    pool = ref.Pool(WeightFormat.Q8, 2, page, 4)
    cache = upload(pool)
    x = rng.standard_normal((T, 4, D)).astype(np.float32)
    x[7, 2:, 3], x[9, 2:, 40], x[59, 2:, 100] = 65504, -65500, 65469
    x[11, 2:, 64:96] = np.where(np.arange(32) % 2, -65504, 65504)
    slots = np.arange(T, dtype=np.int32)
    cache.store(dev(x), T, dev(slots))
    after = download(cache, pool)
    values = after.values(1, slots)
    assert values[7, :, 3].max() == 65532 and np.abs(values - x[:, 2:]).max() <= 516 / 2
    for type_ in TYPES:
        v = dev(np.zeros((T, 2, D), NP[type_]))
        cache.load(dev(slots), T, None, v, type=type_)
        with np.errstate(over="ignore"):
            assert np.array_equal(v.to_array(NP[type_], (T, 2, D)), values.astype(NP[type_]))
    table = np.arange(4, dtype=np.int32)[None]
    for type_ in TYPES:
        for m in (1, 6, 40):
            q = (0.1 * rng.standard_normal((m, 4, D))).astype(NP[type_])
            got = run_attention(after, q, (m,), (T,), table, type_, cache=cache)
            of_sequences(after, q, (m,), (T,), table, got, type_=type_)


@pytest.mark.parametrize("size", [516.0, -516.0, 3000.0, 65504.0])
def test_q8_values_beyond_fp16_in_chunks_of_fp32_queries(size):
    q8_values_beyond_fp16(paged.F32, 40, size)


@pytest.mark.parametrize("where", ["later", "light"])
@pytest.mark.parametrize("m", [5, 60])
def test_large_values_leave_rows_exact_that_do_not_see_them(m, where):
    """fp32 queries over small q8 values: a value of 65504 at a later token, or a large one at a slot of next to no
    weight, takes nothing from the accuracy of a row."""
    rng = np.random.default_rng(57)
    kv = 126
    pool, table = filled(WeightFormat.Q8, 2, 16, (kv,), rng)
    pool.scales[0][:] = np.where(np.isnan(pool.scales[0]), np.nan, 1e-3)
    pool.scales[1][:] = np.where(np.isnan(pool.scales[1]), np.nan, 1e-4 * rng.uniform(0.6, 1, pool.scales[1].shape))
    if where == "later":
        pool.scales[1][table[0, (kv - 1) // 16], :, (kv - 1) % 16] = 516
    else:
        at = table[0, 4], slice(None), 3  # slot 67, a score of -60 log 2
        pool.data[0][at], pool.scales[0][at], pool.scales[1][at] = -127, 60 * np.log(2) / (4 * 127 * D ** 0.5), 500
    q = (4 + 0.1 * rng.standard_normal((m, 4, D))).astype(np.float32)
    got = run_attention(pool, q, (m,), (kv,), table, paged.F32)
    of_sequences(pool, q, (m,), (kv,), table, got)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m", [1, 40])
@pytest.mark.parametrize("size,weight", [(1e-2, 12), (1e-4, 17), (1e-4, 20), (3e-5, 17), (3e-5, 20)])
def test_small_values_behind_a_slot_that_takes_the_weight(fmt, type_, m, size, weight):
    """A first slot of value zero has nearly all of every softmax; what the 2^-12 to 2^-20 weights of the others
    give has its own size's accuracy, also where V is small."""
    rng = np.random.default_rng(54)
    kv, page = 2000, 64
    pool, table = filled(fmt, 2, page, (kv,), rng)
    first = table[0, 0], slice(None), 0
    if pool.q8:
        pool.scales[0][:] = np.where(np.isnan(pool.scales[0]), np.nan, 1e-3)
        pool.scales[1][:] = np.where(np.isnan(pool.scales[1]), np.nan, size * rng.uniform(0.6, 1, pool.scales[1].shape))
        pool.data[0][first], pool.scales[0][first], pool.scales[1][first] = 127, weight * np.log(2) / (4 * 127 * D ** 0.5), 0
    else:
        pool.data[0][:] = pool.data[0] * np.float16(0.1)
        pool.data[1][:] = pool.data[1] * np.float16(size * 60)
        pool.data[0][first], pool.data[1][first] = weight * np.log(2) / (4 * D ** 0.5), 0
    q = (4 + 0.1 * rng.standard_normal((m, 4, D))).astype(NP[type_])
    got = run_attention(pool, q, (m,), (kv,), table, type_)
    # fp16 outputs below 2^-14 step by 2^-24: half a step, spread evenly.
    of_sequences(pool, q, (m,), (kv,), table, got, floor=2.0 ** -25 if type_ == paged.F16 else 0.0, type_=type_)


@pytest.mark.parametrize("size", [516.0, -516.0, 3000.0, 65504.0])
def test_q8_values_beyond_fp16_in_chunks_of_fp16_queries(size):
    q8_values_beyond_fp16(paged.F16, 40, size)


@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_values_of_all_sizes_along_a_sequence(order):
    """fp16 queries, a prompt over q8 values whose size changes by factors of up to 2^13 from 64 slots to the next,
    and among the 16-slot tiles of one: rows are as exact as their outputs' size asks."""
    rng = np.random.default_rng(58)
    kv, m = 640, 600
    pool, table = filled(WeightFormat.Q8, 1, 64, (kv,), rng)
    p = np.arange(kv)
    size = {"rising": 2.0 ** (p // 64 * 1.4 - 13), "falling": 2.0 ** (1 - p // 64 * 1.4), "mixed": 2.0 ** -(p // 16 * 5 % 12)}[order]
    w = pool.where(pool_slots(pool, table[0], kv))
    pool.scales[1][w] = (size[:, None, None] * rng.uniform(0.6, 1, (kv, 1, 4))).astype(np.float16)
    q = (0.5 * rng.standard_normal((m, 2, D))).astype(np.float16)
    got = run_attention(pool, q, (m,), (kv,), table, paged.F16)
    of_sequences(pool, q, (m,), (kv,), table, got, floor=2.0 ** -25, type_=paged.F16)


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("fmt", FMTS)
def test_stored_rows_that_are_no_numbers_stay_so(fmt, what):
    """A key or value that is no number is none in the pool either: the value itself (f16), its group (q8)."""
    rng = np.random.default_rng(55)
    pool = ref.Pool(fmt, 2, 16, 1)
    cache = upload(pool)
    x = rng.standard_normal((5, 4, D)).astype(np.float32)
    x[1, 0, 40], x[3, 3, 127] = what, what
    slots = np.arange(5, dtype=np.int32)
    cache.store(dev(x), 5, dev(slots))
    k, v = (dev(np.zeros((5, 2, D), np.float32)) for _ in range(2))
    cache.load(dev(slots), 5, k, v)
    got = np.concatenate([b.to_array(np.float32, (5, 2, D)) for b in (k, v)], 1)  # [token][k heads, v heads]
    width = 32 if pool.q8 else 1
    spoiled = np.zeros(got.shape, bool)
    spoiled[1, 0, 40 // width * width:40 // width * width + width] = True
    spoiled[3, 3, 127 // width * width:128] = True
    assert not np.isfinite(got[spoiled]).any()
    off = np.abs(np.where(spoiled, 0, got) - np.where(spoiled, 0, x))
    assert np.abs(x[~spoiled]).max() < 4.5  # q8: half a step of a scale that is one fp16 step above 4.5 / 127 at most
    assert (off <= np.where(spoiled, 0, np.abs(x)) * 2.0 ** -11 + (4.5 / 254 * (1 + 2.0 ** -9) if pool.q8 else 0))[~spoiled].all()


@pytest.mark.parametrize("fmt", FMTS)
def test_chunks_among_hundreds_of_sequences(fmt):
    """Chunks are found behind runs of more than 64 sequences that have none, many of them of one length."""
    rng = np.random.default_rng(38)
    q_lens = [1] * 70 + [20] * 90 + [2] * 130 + [0] * 20 + [30, 1, 80]
    kv_lens = [int(x) for x in rng.integers(1, 40, 70)] + [33] * 90 + [int(x) for x in rng.integers(2, 50, 150)] + [30, 200, 100]
    pool, table = filled(fmt, 2, 16, kv_lens, rng)
    q = rng.standard_normal((sum(q_lens), 2, D)).astype(np.float32)
    got = run_attention(pool, q, q_lens, kv_lens, table, paged.F32)
    want, reach, vmax = ref.attention(pool, q, q_lens, kv_lens, table)
    assert np.abs(got - want).max() <= ref.attention_tol(False, pool.q8, reach, vmax)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m", [1, 7, 40, 130])
@pytest.mark.parametrize("spread", [0.05, 1.0, 4.0])
def test_attention_error_in_root_mean_square(fmt, type_, m, spread):
    """Scores of this rms; single tokens, drafts and chunks, every row by itself and all together."""
    rng = np.random.default_rng(56)
    q_lens, kv_lens = (m, 1, m), (601, 333, 200)
    pool, table = filled(fmt, 2, 16, kv_lens, rng)
    q = rng.standard_normal((2 * m + 1, 4, D))
    size = np.sqrt(np.mean([np.mean(pool.values(0, pool_slots(pool, t, n)) ** 2) for t, n in zip(table, kv_lens)]))
    q = (q * spread / size).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_)
    of_sequences(pool, q, q_lens, kv_lens, table, got, type_=type_)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m", [1, 20])
def test_attention_error_over_a_long_sequence(fmt, type_, m):
    """The same where many workgroups share the slots and their partials are joined."""
    rng = np.random.default_rng(59)
    kv = 9001
    pool, table = filled(fmt, 1, 64, (kv,), rng)
    q = (rng.standard_normal((m, 2, D)) / np.sqrt(np.mean(pool.values(0, pool_slots(pool, table[0], kv)) ** 2))).astype(NP[type_])
    got = run_attention(pool, q, (m,), (kv,), table, type_)
    of_sequences(pool, q, (m,), (kv,), table, got, type_=type_)


def pool_slots(pool, row, n):
    p = np.arange(n)
    return row[p // pool.page].astype(np.int64) * pool.page + p % pool.page


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m", [1, 20])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_values_that_are_no_numbers_where_workgroups_join(fmt, type_, m, what):
    """A slot whose weight, e^-200, is nothing in fp32, in another workgroup's share than the slot that has it all:
    the rows that see it give no number, as they do where one workgroup has both."""
    rng = np.random.default_rng(60)
    kv = 3000
    pool, table = filled(fmt, 1, 64, (kv,), rng)
    first, far = (table[0, 0], slice(None), 0), (table[0, 2500 // 64], slice(None), 2500 % 64)
    if pool.q8:
        pool.scales[0][:] = np.where(np.isnan(pool.scales[0]), np.nan, 1e-3)
        pool.data[0][first], pool.scales[0][first] = 127, 200 / (4 * 127 * D ** 0.5)
        pool.scales[1][far][..., 1] = what
    else:
        pool.data[0][:] = pool.data[0] * np.float16(0.1)
        pool.data[0][first] = 200 / (4 * D ** 0.5)
        pool.data[1][far][..., 37] = what
    q = (4 + 0.1 * rng.standard_normal((m, 2, D))).astype(NP[type_])
    got = run_attention(pool, q, (m,), (kv,), table, type_)
    spoiled = np.zeros(D, bool)
    spoiled[slice(32, 64) if pool.q8 else 37] = True
    assert not np.isfinite(got[..., spoiled]).any() and np.isfinite(got[..., ~spoiled]).all()
