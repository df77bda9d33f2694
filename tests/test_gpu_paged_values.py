"""GPU tests of the operators on paged K/V caches where the values are unusual.  Definitions in paged_ref.py."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_ref as ref  # noqa: E402
from instantcua_amd import paged  # noqa: E402
from test_gpu_paged import D, FMTS, NP, TYPES, filled, run_attention  # noqa: E402

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
