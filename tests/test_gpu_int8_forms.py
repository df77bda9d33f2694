"""GPU tests of every form of the products on 8-bit integers with more steps than it has stages, and of sums that pass
2^30 on the way to small results, which fp32 shows to the unit."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from instantcua_amd import int8  # noqa: E402
from int8_shapes import DEEP  # noqa: E402
from test_gpu_int8 import run_matmul, test_matmul as matmul_against_float64  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", [int8.F32, int8.F16])
@pytest.mark.parametrize("form,gated,m,n,k", DEEP)
def test_deep(type, form, gated, m, n, k):
    for kind, gap in [("gated", 1)] if gated else [("plain", 0), ("add", 3)]:
        matmul_against_float64(type, kind, m, n, k, gap)


@pytest.mark.parametrize("form,gated,m,n,k", DEEP)
def test_sums_to_the_unit(form, gated, m, n, k):
    """Half of the products are 127^2, the other half as much less, in an order of their own for every channel: partial
    sums are as large as half the depth allows, and a sum is what the first code, 1 in x, and some left-over codes
    make it.  With scales of one, fp32 holds sums below 2^24 exactly; a gate of 64 passes 64 times the up."""
    rng = np.random.default_rng(k)
    x = np.full((m, k), 127, np.int8)
    x[:, 0], x[1::2, 1:] = 1, -127
    w = np.full((n * (1 + gated), k), 127, np.int8)
    half = (k - 1) // 2
    w[::2, 1:1 + half], w[1::2, 1 + half:1 + 2 * half] = -127, -127
    w[:, 0], w[:, 1 + 2 * half:] = rng.integers(-127, 128, len(w)), 0
    w[:, 2 * half] = w[:, 2 * half] // 127 * rng.integers(120, 128, len(w))
    if gated:
        w[:n, 2 * half] = np.where(w[:n, 2 * half] > 0, 127, -127)
        w[:n, 0] = 64
    sums = x.astype(np.float64) @ w.astype(np.float64).T
    assert np.abs(sums).max() < 2 ** 16 and len(np.unique(sums)) > 60
    got = run_matmul(x, np.ones(m, np.float32), w, np.ones(len(w), np.float32), gated=bool(gated))
    # 1 + exp(-64) is 1 in fp32, and its inverse by the instruction, too, or a step of 2^-23 from it.
    if gated:
        assert (sums[:, :n] == 64).all()
        want = 64 * sums[:, n:]
        assert (np.abs(got - want) <= 2.0 ** -23 * np.abs(want)).all()
    else:
        assert np.array_equal(got, sums)


@pytest.mark.parametrize("m", [1, 20, 150])
def test_sums_to_the_unit_at_the_largest_depth(m):
    """2^17 codes: 2^16 products of 127^2 of one sign, partial sums of 2^30, before those of the other."""
    k, n = 1 << 17, 40
    x = np.full((m, k), 127, np.int8)
    w = np.full((n, k), 127, np.int8)
    w[::2, :k // 2], w[1::2, k // 2:] = -127, -127
    x[:, 5], w[:, 5] = 1, np.arange(n)
    sums = x.astype(np.float64) @ w.astype(np.float64).T
    assert np.abs(sums).max() < 2 ** 24 and len(np.unique(sums)) == n
    assert np.array_equal(run_matmul(x, np.ones(m, np.float32), w, np.ones(n, np.float32)), sums)
