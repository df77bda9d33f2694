"""GPU tests of the attention over paged caches with a window and first slots, and with shared prefixes, against
float64 definitions: windows and prefixes next to every step of the kernels, slots that no token sees holding NaN,
pages given back, sequences without tokens, shorter than their prefix, in no group."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_bounds as bounds  # noqa: E402
import paged_forms_ref as forms  # noqa: E402
import paged_ref as ref  # noqa: E402
from instantcua_amd import paged  # noqa: E402
from instantcua_amd.modelfile import WeightFormat  # noqa: E402
from test_gpu_paged import D, FMTS, NP, TYPES, dev, filled, run_attention, tables_of, upload  # noqa: E402

pytestmark = pytest.mark.gpu


class Form:
    """The cache, with `attention` and `attention_work` of a form, so that both are called alike."""

    def __init__(self, pool, cache=None, **kw):
        self.cache, self.kw = cache or upload(pool), kw

    def attention_work(self, heads, n_seqs, n_tokens, **kw):
        if "window" in self.kw:
            return self.cache.attention_window_work(heads, n_seqs, n_tokens, self.kw["window"], self.kw["sinks"], **kw)
        return self.cache.attention_prefix_work(heads, n_seqs, n_tokens, len(self.kw["lens"]), self.kw.get("max_prefix", 0), **kw)

    def attention(self, q, out, heads, start, kv, table, n_seqs, n_tokens, width, **kw):
        if "window" in self.kw:
            self.cache.attention_window(q, out, heads, start, kv, table, n_seqs, n_tokens, width, self.kw["window"],
                                        self.kw["sinks"], **kw)
        else:
            g = [dev(np.asarray(a, np.int32)) for a in (self.kw["starts"], self.kw["lens"])]
            self.cache.attention_prefix(q, out, heads, start, kv, table, n_seqs, n_tokens, width, *g, len(self.kw["lens"]),
                                        self.kw.get("max_prefix", 0), **kw)


def check(pool, q, q_lens, kv_lens, table, got, type_, window=None, sinks=0, chunk=None, want_pool=None, table_ref=None):
    """Every row against the definition, largest error and root mean square."""
    want, reach, vmax = forms.attention(want_pool or pool, q, q_lens, kv_lens, table if table_ref is None else table_ref, window, sinks)
    fp16 = type_ == paged.F16
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= ref.attention_tol(fp16, pool.q8, reach, vmax)
    group = q.shape[1] // pool.n_kv
    chunk = any(bounds.chunked(m, group) for m in q_lens) if chunk is None else chunk
    n = max(kv_lens)
    # One more rounding step for the join of a row's two parts is within the joins that the bound counts.
    bounds.check(got, want, bounds.rms_bound(fp16, pool.q8, chunk, reach, n))


# ---------------------------------------------------------------------------------------------
# window

def windowed(fmt, n_kv, page, q_lens, kv_lens, window, sinks, rng):
    """A pool where slots that no token sees hold NaN, and pages without any that is seen are given back (any number
    outside the pool)."""
    table, pages = tables_of(kv_lens, page, rng)
    pool = ref.Pool(fmt, n_kv, page, pages)
    for s, (m, n) in enumerate(zip(q_lens, kv_lens)):
        own = (n - m + np.arange(m))[:, None]
        p = np.nonzero(forms.seen(own, n, window, sinks).any(0))[0] if m else np.arange(0)
        pool.fill(table[s, p // page].astype(np.int64) * page + p % page, rng)
        gone = np.setdiff1d(np.arange(table.shape[1]), p // page)
        table[s, gone] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31], gone.size)
    return pool, table


WINDOWS = [
    # heads, n_kv, page, [(new tokens, slots)]
    (16, 8, 64, [(1, 1)]),
    (16, 8, 64, [(1, 2000), (1, 17), (1, 64), (1, 130), (0, 300), (1, 0), (1, 33)]),
    (16, 8, 16, [(8, 1700), (3, 3), (5, 100)]),
    (16, 8, 48, [(9, 9), (1, 250), (41, 900)]),
    (4, 4, 32, [(20, 400), (16, 16), (17, 40), (1, 1000)]),
    (12, 4, 16, [(6, 90), (1, 31), (30, 33)]),
    (16, 1, 16, [(1, 700), (7, 200)]),
    (6, 2, 32, [(5, 2), (3, 0), (2, 40)]),
    (2, 2, 16, [(150, 1333), (1, 40)]),
    (16, 8, 64, [(300, 300)]),
]
SIZES = [(1, 0), (1, 1), (5, 4), (16, 0), (31, 33), (32, 64), (33, 1), (100, 16), (127, 128), (128, 129), (300, 200),
         (2 ** 31 - 1, 0), (40, 2 ** 31 - 1)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("case", range(len(WINDOWS)))
def test_window(fmt, type_, case):
    heads, n_kv, page, lens = WINDOWS[case]
    q_lens, kv_lens = zip(*lens)
    for i, (window, sinks) in enumerate(SIZES):
        rng = np.random.default_rng(1000 * case + i)
        pool, table = windowed(fmt, n_kv, page, q_lens, kv_lens, window, sinks, rng)
        q = (rng.standard_normal((sum(q_lens), heads, D)) * 1.5).astype(NP[type_])
        got = run_attention(pool, q, q_lens, kv_lens, table, type_, extra=case % 3, cache=Form(pool, window=window, sinks=sinks))
        print(case, window, sinks, flush=True)
        check(pool, q, q_lens, kv_lens, table, got, type_, window, sinks)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("q_lens,kv_lens,window,sinks", [
    ((1,) * 5, (9000, 4097, 5000, 300, 8191), 4096, 4), ((1, 1), (30000, 20000), 100, 10000),
    ((700, 1, 300), (5000, 7000, 300), 1000, 130), ((2000,), (2500,), 130, 0), ((12, 5), (6000, 2000), 2047, 3),
])
def test_window_of_long_sequences(fmt, type_, q_lens, kv_lens, window, sinks):
    """Windows that several workgroups share, and tiles whose rows' windows begin in different steps."""
    rng = np.random.default_rng(len(q_lens) + window)
    pool, table = windowed(fmt, 2, 64, q_lens, kv_lens, window, sinks, rng)
    q = (rng.standard_normal((sum(q_lens), 4, D)) * 1.5).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, cache=Form(pool, window=window, sinks=sinks))
    check(pool, q, q_lens, kv_lens, table, got, type_, window, sinks)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("heads,n_kv,q_lens,kv_lens", [
    (64, 64, (1, 1, 1, 1), (700, 65, 1, 400)),                                # 256 pairs: a workgroup of eight waves each
    (128, 64, (3, 0, 8, 1), (300, 200, 500, 0)),
    (128, 64, (1, 2, 1, 1, 8, 1, 0, 1), (300, 90, 64, 1000, 450, 33, 20, 2)),  # 512: of four
    (72, 72, (1,) * 12, tuple(range(100, 700, 50))),                          # 864: two rounds
])
def test_windows_that_fill_the_gpu(fmt, type_, heads, n_kv, q_lens, kv_lens):
    """Sequences whole in one workgroup each."""
    for window, sinks in ((200, 5), (33, 0), (64, 64)):
        rng = np.random.default_rng(window)
        pool, table = windowed(fmt, n_kv, 16, q_lens, kv_lens, window, sinks, rng)
        form = Form(pool, window=window, sinks=sinks)
        assert form.attention_work(heads, len(q_lens), sum(q_lens), max_q=max(q_lens), max_kv=max(kv_lens)) == 0
        q = (rng.standard_normal((sum(q_lens), heads, D)) * 1.5).astype(NP[type_])
        got = run_attention(pool, q, q_lens, kv_lens, table, type_, cache=form)
        check(pool, q, q_lens, kv_lens, table, got, type_, window, sinks)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("window,sinks", [(40, 3), (200, 0), (700, 70)])
def test_windows_of_many_sequences_beside_chunks(fmt, type_, window, sinks):
    """Single tokens, drafts, chunks and sequences without tokens, more than a wave looks at, in any order."""
    rng = np.random.default_rng(window)
    q_lens = tuple(int(m) for m in rng.choice([1, 1, 1, 0, 5, 8, 9, 40], 150))
    kv_lens = tuple(int(m + rng.integers(0, 900)) for m in q_lens)
    pool, table = windowed(fmt, 2, 32, q_lens, kv_lens, window, sinks, rng)
    q = rng.standard_normal((sum(q_lens), 4, D)).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, extra=2, cache=Form(pool, window=window, sinks=sinks))
    check(pool, q, q_lens, kv_lens, table, got, type_, window, sinks)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
def test_a_window_of_everything_is_the_plain_attention(fmt, type_):
    """To the bit: the same slots in the same steps."""
    rng = np.random.default_rng(5)
    q_lens, kv_lens = (1, 40, 3, 200), (1500, 700, 900, 200)
    pool, table = filled(fmt, 8, 64, kv_lens, rng)
    q = rng.standard_normal((sum(q_lens), 16, D)).astype(NP[type_])
    cache = upload(pool)
    want = run_attention(pool, q, q_lens, kv_lens, table, type_, cache=cache)
    for window, sinks in ((1500, 0), (2 ** 31 - 1, 7), (3, 1500), (1499, 1)):
        assert np.array_equal(run_attention(pool, q, q_lens, kv_lens, table, type_, cache=Form(pool, cache, window=window, sinks=sinks)), want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("m,kv", [(6, 400), (60, 700), (100, 500)])
def test_values_of_a_window_that_are_no_numbers(fmt, type_, what, m, kv):
    """V of one slot is spoiled: rows whose window has it, or for which it is one of the first, give no number in
    those dims; every other row and dim what it gives without."""
    rng = np.random.default_rng(m)
    window, sinks = 37, 3
    q_lens, kv_lens = (m, 3), (kv, 40)
    pool, table = windowed(fmt, 2, 16, q_lens, kv_lens, window, sinks, rng)
    q = rng.standard_normal((m + 3, 4, D)).astype(NP[type_])
    want, reach, vmax = forms.attention(pool, q, q_lens, kv_lens, table, window, sinks)
    tol = ref.attention_tol(type_ == paged.F16, pool.q8, reach, vmax)
    for slot in (1, kv - m - window + 1, kv - m - 3, kv - m // 2, kv - 1):
        at = table[0, slot // 16], 1, slot % 16
        dims = slice(64, 96) if pool.q8 else slice(37, 38)
        store = pool.scales[1][at] if pool.q8 else pool.data[1][at]
        kept = store.copy()
        store[2 if pool.q8 else 37] = what
        got = run_attention(pool, q, q_lens, kv_lens, table, type_, cache=Form(pool, window=window, sinks=sinks))
        own = kv - m + np.arange(m)
        sees = np.zeros(got.shape, bool)
        rows = np.nonzero(forms.seen(own[:, None], kv, window, sinks)[:, slot])[0]
        sees[rows[:, None], np.array([2, 3]), dims] = True
        assert not np.isfinite(got[sees]).any() and sees.any(), slot
        assert np.abs(got - want)[~sees].max() <= tol, slot
        store[:] = kept


# ---------------------------------------------------------------------------------------------
# shared prefixes

def shared(fmt, n_kv, page, kv_lens, starts, lens, rng):
    """Tables where a group's sequences have the whole pages of its prefix in common, and copies of a page that is
    the prefix's in part."""
    table, pages = tables_of([max(n, 1) for n in kv_lens], page, rng)
    pool = ref.Pool(fmt, n_kv, page, pages)
    for g, P in enumerate(lens):
        a, b = starts[g], starts[g + 1]
        for s in range(a, b):
            table[s, :min(P, kv_lens[s]) // page] = table[a, :min(P, kv_lens[s]) // page]
    for s, n in enumerate(kv_lens):
        p = np.arange(n)
        pool.fill(table[s, p // page].astype(np.int64) * page + p % page, rng)
    for g, P in enumerate(lens):
        for s in range(starts[g], starts[g + 1]):
            for p in range(min(P, kv_lens[s]) // page * page, min(P, kv_lens[s], kv_lens[starts[g]])):
                for i in range(2):
                    for x in (pool.data, pool.scales):
                        x[i][table[s, p // page], :, p % page] = x[i][table[starts[g], p // page], :, p % page]
    return pool, table


PREFIXES = [
    # heads, n_kv, page, [(new tokens, slots)], groups' starts, prefixes
    (16, 8, 64, [(1, 300), (1, 260)], [0, 2], [256]),
    (16, 8, 64, [(1, 300), (1, 260), (1, 700), (1, 257)], [0, 4], [256]),
    (16, 8, 16, [(1, 500)] * 9, [0, 9], [499]),                      # 18 rows of the prefix: the other kernel
    (16, 8, 64, [(1, 200 + 7 * i) for i in range(70)], [0, 70], [192]),  # 140 rows: two tiles, more than 64 spans
    (4, 4, 32, [(3, 300), (5, 290), (1, 900), (2, 257)], [0, 4], [256]),
    (16, 8, 48, [(1, 400), (1, 300), (1, 500), (1, 600), (1, 20), (1, 450)], [1, 3, 4, 6], [250, 400, 300]),  # one of one
    (12, 4, 16, [(40, 400), (1, 300), (30, 310), (0, 256), (7, 1000)], [0, 5], [256]),
    (16, 1, 16, [(1, 700), (7, 650), (2, 641)], [0, 3], [640]),
    (16, 8, 64, [(100, 900), (60, 460), (1, 400), (1, 2000)], [0, 3], [390]),
    (2, 2, 16, [(150, 1333), (100, 1000), (1, 40), (1, 900), (1, 901)], [0, 2, 2, 3, 5], [900, 500, 30, 880]),
    (6, 2, 32, [(2, 300), (1, 290), (4, 280)], [0, 3], [127]),       # less than a step: nothing is shared
    (8, 8, 128, [(1, 1000), (1, 3000), (20, 2500)], [0, 3], [900]),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("case", range(len(PREFIXES)))
def test_prefix(fmt, type_, case):
    heads, n_kv, page, lens, starts, prefixes = PREFIXES[case]
    q_lens, kv_lens = zip(*lens)
    rng = np.random.default_rng(300 + case)
    pool, table = shared(fmt, n_kv, page, kv_lens, starts, prefixes, rng)
    q = (rng.standard_normal((sum(q_lens), heads, D)) * 1.5).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, extra=case % 3, cache=Form(pool, starts=starts, lens=prefixes))
    check(pool, q, q_lens, kv_lens, table, got, type_, chunk=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
def test_the_prefix_is_read_through_the_first_table(fmt, type_):
    """The other sequences' table entries for it may be anything; up to the last whole 128 slots it holds nothing
    else."""
    rng = np.random.default_rng(6)
    for q_lens, kv_lens in (((1, 1, 1), (400, 500, 385)), ((20, 1, 50), (420, 500, 440)), ((1,) * 12, (390,) * 12)):
        starts, prefixes = [0, len(q_lens)], [384]
        pool, table = shared(fmt, 2, 64, kv_lens, starts, prefixes, rng)
        q = rng.standard_normal((sum(q_lens), 4, D)).astype(NP[type_])
        spoiled = table.copy()
        spoiled[1:, :6] = rng.choice([-1, pool.n_pages, -2 ** 31, 2 ** 31 - 1], spoiled[1:, :6].shape)
        got = run_attention(pool, q, q_lens, kv_lens, spoiled, type_, cache=Form(pool, starts=starts, lens=prefixes))
        check(pool, q, q_lens, kv_lens, table, got, type_, chunk=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens,P", [
    ([(1, 600), (1, 300), (1, 512), (1, 511), (1, 0), (1, 513)], 512),     # shorter than the prefix, by one, and empty
    ([(1, 600)] * 10 + [(1, 0), (1, 1), (1, 100), (1, 400)], 512),
    ([(40, 600), (600, 600), (30, 520), (5, 100), (3, 2)], 512),           # tokens of the prefix itself
    ([(1, 700), (8, 515), (2, 640)], 512),                                 # a draft that begins in it
])
def test_tokens_that_do_not_see_all_of_the_prefix(fmt, type_, lens, P):
    q_lens, kv_lens = zip(*lens)
    rng = np.random.default_rng(len(lens))
    starts, prefixes = [0, len(lens)], [P]
    pool, table = shared(fmt, 2, 64, kv_lens, starts, prefixes, rng)
    q = rng.standard_normal((sum(q_lens), 4, D)).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, cache=Form(pool, starts=starts, lens=prefixes))
    check(pool, q, q_lens, kv_lens, table, got, type_, chunk=True)


def test_prefixes_longer_than_their_bound_and_groups_outside_the_batch():
    """Nothing outside the buffers is read or written; where sequences do share their slots, the outputs are right."""
    rng = np.random.default_rng(8)
    q_lens, kv_lens = (1,) * 6, (700, 720, 650, 800, 650, 641)
    pool, table = shared(WeightFormat.F16, 2, 32, kv_lens, [0, 6], [640], rng)
    q = rng.standard_normal((6, 4, D)).astype(np.float32)
    for starts, prefixes, bound in (([0, 6], [10 ** 9], 640), ([-5, 3, 10 ** 9], [640, 600], 0), ([0, 6], [-1], 640),
                                    ([0, 6], [2 ** 31 - 1], 300), ([2 ** 31 - 1, 2 ** 31 - 1], [640], 0), ([0, 6], [640], 64)):
        form = Form(pool, starts=starts, lens=prefixes, max_prefix=bound)
        got = run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=form)
        check(pool, q, q_lens, kv_lens, table, got, paged.F32, chunk=True)


def test_groups_that_do_not_rise_stay_inside_the_buffers():
    rng = np.random.default_rng(9)
    q_lens, kv_lens = (1, 20, 1, 1, 30, 1), (700, 720, 650, 800, 690, 641)
    pool, table = shared(WeightFormat.Q8, 2, 32, kv_lens, [0, 6], [640], rng)
    q = rng.standard_normal((sum(q_lens), 4, D)).astype(np.float32)
    for starts in ([6, 0, 6], [4, 2, 5, 0, 6], [0, 6, 0, 6, 0, 6]):
        run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=Form(pool, starts=starts, lens=[640] * (len(starts) - 1)))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("seqs,m,prefix,own", [(64, 1, 4096, 300), (40, 4, 2900, 1000), (5, 200, 1500, 1200), (3, 1, 9000, 3000), (200, 1, 640, 64)])
def test_prefix_of_long_sequences(fmt, type_, seqs, m, prefix, own):
    """Prefixes and sequences that several workgroups share."""
    rng = np.random.default_rng(seqs)
    q_lens = [m if i % 3 else max(1, m - i % 5) for i in range(seqs)]
    kv_lens = [prefix + int(rng.integers(a, own + 1)) for a in q_lens]
    starts, prefixes = [0, seqs // 3, seqs], [prefix, prefix - 200]
    pool, table = shared(fmt, 1, 64, kv_lens, starts, prefixes, rng)
    q = (rng.standard_normal((sum(q_lens), 2, D)) * 1.5).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, cache=Form(pool, starts=starts, lens=prefixes))
    check(pool, q, q_lens, kv_lens, table, got, type_, chunk=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("m", [1, 9])
def test_values_of_a_prefix_that_are_no_numbers(fmt, what, m):
    """They spoil every token of the group, and those of an own slot only their sequence."""
    rng = np.random.default_rng(m)
    q_lens, kv_lens = (m,) * 4, (300, 320, 400, 290)
    for slot, rows in ((17, slice(0, 3 * m)), (310, slice(m, 2 * m))):
        pool, table = shared(fmt, 2, 16, kv_lens, [0, 3], [256], rng)
        q = rng.standard_normal((4 * m, 4, D)).astype(np.float32)
        want, reach, vmax = forms.attention(pool, q, q_lens, kv_lens, table)
        s = 1 if slot == 310 else 0
        at = table[s, slot // 16], 1, slot % 16
        dims = slice(64, 96) if pool.q8 else slice(37, 38)
        (pool.scales[1][at] if pool.q8 else pool.data[1][at])[2 if pool.q8 else 37] = what
        got = run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=Form(pool, starts=[0, 3], lens=[256]))
        sees = np.zeros(got.shape, bool)
        sees[rows, 2:, dims] = True
        if slot == 310:
            sees[m:m + max(0, 310 - (320 - m))] = False
        assert not np.isfinite(got[sees]).any()
        assert np.abs(got - want)[~sees].max() <= ref.attention_tol(False, pool.q8, reach, vmax)


def test_prefix_repeats_to_the_bit():
    rng = np.random.default_rng(12)
    q_lens, kv_lens = (1, 1, 40, 1), (1500, 700, 900, 640)
    pool, table = shared(WeightFormat.Q8, 8, 64, kv_lens, [0, 4], [600], rng)
    q = rng.standard_normal((43, 16, D)).astype(np.float32)
    form = Form(pool, starts=[0, 4], lens=[600])
    first = run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=form)
    for _ in range(3):
        assert np.array_equal(run_attention(pool, q, q_lens, kv_lens, table, paged.F32, cache=form), first)
