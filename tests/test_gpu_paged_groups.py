"""GPU tests of attention with shared prefixes in as many groups as a call takes, and where a group's first sequence
does not hold its prefix, against the float64 definition: idle places, sessions that are still to get the prefix,
tables with other sequences' pages behind the slots in use."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as ref  # noqa: E402
from test_gpu_paged import D, FMTS, NP, TYPES, run_attention, tables_of  # noqa: E402
from test_gpu_paged_forms import Form, check  # noqa: E402

pytestmark = pytest.mark.gpu


def grouped(fmt, n_kv, page, kv_lens, starts, lens, rng):
    """Tables where a group's sequences have the pages of its prefix in common, as far as they have slots; entries
    behind those are any other pages."""
    table, pages = tables_of([max(n, 1) for n in kv_lens], page, rng)
    pool = ref.Pool(fmt, n_kv, page, pages)
    common = [0] * len(kv_lens)
    leader = list(range(len(kv_lens)))
    for g, P in enumerate(lens):
        a, b = starts[g], starts[g + 1]
        for s in range(a, b):
            leader[s], common[s] = a + int(np.argmax(kv_lens[a:b])), min(P, kv_lens[s])
            table[s, :common[s] // page] = table[leader[s], :common[s] // page]
    for s, n in enumerate(kv_lens):
        p = np.arange(n)
        pool.fill(table[s, p // page].astype(np.int64) * page + p % page, rng)
    for s, l in enumerate(leader):  # a page that is the prefix's in part
        for p in range(common[s] // page * page, common[s]):
            for x in (*pool.data, *pool.scales) if pool.q8 else pool.data:
                x[table[s, p // page], :, p % page] = x[table[l, p // page], :, p % page]
        behind = -(-kv_lens[s] // page)
        table[s, behind:] = rng.integers(0, pages, table.shape[1] - behind)
    return pool, table


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens,starts,prefixes", [
    ([(0, 0), (1, 600), (1, 700), (1, 530)], [0, 4], [512]),                     # an idle place
    ([(0, 0), (0, 0)] + [(1, 600)] * 10, [0, 12], [512]),
    ([(1, 300), (1, 600), (1, 513)], [0, 3], [512]),                             # shorter, with tokens of its own
    ([(1, 511), (1, 600), (8, 900)], [0, 3], [512]),                             # by one slot
    ([(40, 200), (30, 600), (1, 520), (100, 700)], [0, 4], [512]),               # a chunk of the prefix itself
    ([(1, 0)] * 70 + [(1, 400), (1, 300), (2, 390)], [0, 73], [384]),            # behind the first 64
    ([(1, 200), (1, 450), (1, 300), (30, 470), (1, 900)], [0, 4], [512]),                  # none has all of it
    ([(0, 0), (1, 0), (3, 2), (1, 900)], [0, 3], [512]),                                   # nor any of it
    ([(0, 0), (1, 300), (1, 290), (1, 100), (1, 700), (9, 680)], [0, 3, 6], [256, 640]),
])
def test_the_first_sequence_lacks_the_prefix(fmt, type_, lens, starts, prefixes):
    q_lens, kv_lens = zip(*lens)
    for heads, n_kv, page in ((4, 2, 64), (6, 2, 16)):
        rng = np.random.default_rng(len(lens) + page)
        pool, table = grouped(fmt, n_kv, page, kv_lens, starts, prefixes, rng)
        q = rng.standard_normal((sum(q_lens), heads, D)).astype(NP[type_])
        got = run_attention(pool, q, q_lens, kv_lens, table, type_, extra=1, cache=Form(pool, starts=starts, lens=prefixes, max_prefix=max(prefixes)))
        check(pool, q, q_lens, kv_lens, table, got, type_, chunk=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n_groups,seqs,q_choice", [(64, 200, [1]), (64, 150, [1, 1, 0, 3, 9, 30]), (33, 140, [1, 8]), (17, 70, [1, 1, 40]), (2, 130, [1, 0, 5]), (63, 64, [1, 2])])
def test_many_groups(fmt, type_, n_groups, seqs, q_choice):
    """Groups of none, one and several sequences, sequences in front of the first and behind the last, of any lengths."""
    rng = np.random.default_rng(n_groups + seqs)
    starts = [int(s) for s in np.sort(rng.integers(2, seqs - 1, n_groups + 1))]
    prefixes = [int(p) for p in rng.choice([100, 128, 200, 256, 300, 400], n_groups)]
    q_lens = [int(m) for m in rng.choice(q_choice, seqs)]
    kv_lens = [int(rng.integers(0, 700)) if rng.random() < 0.3 else int(400 + m + rng.integers(0, 200)) for m in q_lens]
    heads, n_kv, page = (4, 2, 32) if n_groups % 2 else (3, 1, 16)
    pool, table = grouped(fmt, n_kv, page, kv_lens, starts, prefixes, rng)
    q = rng.standard_normal((sum(q_lens), heads, D)).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, extra=2, cache=Form(pool, starts=starts, lens=prefixes, max_prefix=400))
    check(pool, q, q_lens, kv_lens, table, got, type_, chunk=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("what", [60000.0, np.nan, np.inf])
def test_slots_that_no_sequence_of_the_group_has(fmt, type_, what):
    """The prefix is said to be longer than any of them: what the tables' pages hold behind their slots takes no part,
    nor accuracy from what is seen."""
    rng = np.random.default_rng(3)
    q_lens, kv_lens, starts, prefixes = (1, 1, 9, 30, 1), (250, 300, 310, 333, 900), [0, 4], [512]
    pool, table = grouped(fmt, 2, 16, kv_lens, starts, prefixes, rng)
    spare = np.setdiff1d(np.arange(pool.n_pages), np.concatenate([table[s, :-(-n // 16)] for s, n in enumerate(kv_lens)]))
    for s, n in enumerate(kv_lens):
        table[s, -(-n // 16):] = rng.choice(spare)
    for i in range(2):
        if pool.q8:
            pool.data[i][spare], pool.scales[i][spare] = 127, what
        else:
            pool.data[i][spare] = what
    q = rng.standard_normal((sum(q_lens), 4, D)).astype(NP[type_])
    got = run_attention(pool, q, q_lens, kv_lens, table, type_, cache=Form(pool, starts=starts, lens=prefixes, max_prefix=512))
    check(pool, q, q_lens, kv_lens, table, got, type_, chunk=True)
