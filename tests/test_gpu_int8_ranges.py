"""GPU tests of the products on 8-bit integers at the ends of fp32's range: gates and ups of any size together, rows
of zeros, quotients that only exact arithmetic tells from a tie."""
import math
import random

import numpy as np
import pytest

from instantcua_amd import int8
from test_gpu_int8 import quantised, run_matmul, run_quantize

pytestmark = pytest.mark.gpu

NEAR = [5, -5, 0.01, -0.7, -30, 30, -79, 79, 1e-30, -1e-20]
FAR = [-81, -88, -100, -104, -115, -150, -200, 81, 200, 1e20, -1e20]
UPS = [1, -64, 1e-30, 1e-33, 2e-36, -2e-37, 1e-38, 1e-40, 2.0 ** -149, 1e20, 1e30, -3e38]


@pytest.mark.parametrize("m", [1, 20, 150, 1100])
@pytest.mark.parametrize("gates", [NEAR, FAR, NEAR + FAR])
def test_gates_and_ups_of_any_size(m, gates):
    """Sums of one, so that gates and ups are the scales.  The exponent of e = exp(-|g|) is 1.5 |g| 2^-24 off (its
    constant and a rounding), e 2^-23 more (the instruction), 1 + e 2^-24, its inverse 2^-23, three products 2^-24 each:
    1.5 |g| + 8 in all, and two roundings to fp32's smallest step."""
    g, u = (np.asarray(a, np.float32) for a in zip(*[(a, b) for a in gates for b in UPS]))
    n = len(g)
    x, w = np.zeros((m, 32), np.int8), np.zeros((2 * n, 32), np.int8)
    x[:, 3], w[:, 3] = 1, 1
    got = run_matmul(x, np.ones(m, np.float32), w, np.concatenate([g, u]), gated=True)
    a, b = g.astype(np.float64), u.astype(np.float64)
    # exp(-|g|) of these leaves no double but for the largest gates, where the result is zero.
    want = a * np.where(a < 0, np.exp(-np.abs(a)), 1) / (1 + np.exp(-np.abs(a))) * b
    tol = (1.5 * np.abs(np.where(np.abs(a) < 1e3, a, 0)) + 8) * 2.0 ** -24 * np.abs(want) + 2.0 ** -149
    most = float(np.finfo(np.float32).max)
    over = np.abs(want) > most
    assert (np.abs(want[~over]) < most * (1 - 2.0 ** -10)).all()
    assert (got[:, over] == np.sign(want[over]) * np.inf).all()
    err = np.abs(got[:, ~over].astype(np.float64) - want[~over])
    bad = err - tol[~over]
    assert np.isfinite(got[:, ~over]).all() and (bad <= 0).all(), (g[~over][bad.max(0).argmax()], u[~over][bad.max(0).argmax()], float(err.max()))


@pytest.mark.parametrize("m", [1, 150])
def test_gates_and_ups_that_are_no_numbers(m):
    """As the definition has them: g / (1 + exp(-g)) u."""
    inf, nan = np.inf, np.nan
    pairs = [(nan, 1), (1, nan), (inf, 2), (inf, 0), (-inf, 1), (-3, inf), (3, -inf), (0, inf), (-200, inf), (2, 3)]
    g, u = (np.asarray(a, np.float32) for a in zip(*pairs))
    n = len(g)
    x, w = np.zeros((m, 16), np.int8), np.ones((2 * n, 16), np.int8)
    x[:, 0] = 1
    with np.errstate(all="ignore"):
        a = g.astype(np.float64)
        want = a / (1 + np.exp(-a)) * u
    got = run_matmul(x, np.ones(m, np.float32), w, np.concatenate([g, u]), gated=True)
    assert np.array_equal(np.isnan(got), np.broadcast_to(np.isnan(want), got.shape))
    some = np.isinf(want)
    assert (got[:, some] == want[some]).all() and abs(got[0, -1] - want[-1]) < 1e-5


@pytest.mark.parametrize("type", [int8.F32, int8.F16])
@pytest.mark.parametrize("cols", [16, 2064, 6160, 16400])
def test_rows_of_zeros_without_eps(type, cols):
    """Their codes and scales are zero, with and without a norm; other rows need no eps."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((5, cols)).astype(np.float16).astype(np.float32)
    x[1], x[4] = 0, -0.0
    norm = rng.uniform(0.5, 2, cols).astype(np.float32)
    for w in (None, norm):
        codes, scales = run_quantize(x, w, type=type, eps=0.0)
        assert (codes[[1, 4]] == 0).all() and (scales[[1, 4]] == 0).all()
        rest = [0, 2, 3]
        want, s = quantised(x[rest], w, eps=0.0)
        assert np.array_equal(codes[rest], want) and (np.abs(scales[rest] - s) <= s * 2.0 ** -23).all()
    # And through a product: zeros, not values that are no numbers.
    y = run_matmul(codes, scales, np.ones((3, cols), np.int8), np.ones(3, np.float32))
    assert (y[[1, 4]] == 0).all() and np.isfinite(y).all()


def next_to_ties(n, seed):
    """n of (x, norm, largest x, k, off) and the largest's norm: 254 x norm = (2 k + 1) largest + off, of 24-bit numbers
    and |off| of at most 16, so that the quotient 127 x norm / largest is k + 1/2 but for off / (2 largest), 2^-42 or
    less."""
    rng = random.Random(seed)
    top_norm, found = rng.randrange(1 << 23, 1 << 24) | 1, []
    while len(found) < n:
        norm = rng.randrange(1 << 23, 1 << 24) | 1
        for k in range(20, 127):
            p, m = 254 * norm, (2 * k + 1) * top_norm
            g = math.gcd(p, m)
            for off in (i * g for i in (-2, -1, 1, 2) if abs(i) * g <= 16):
                for x in range(off // g * pow(p // g, -1, m // g) % (m // g), 1 << 24, m // g):
                    top = (p * x - off) // m
                    if 1 << 22 <= top < 1 << 24 and x >= 1 << 20:
                        found.append((x, norm, top, k, off))
    return top_norm, found[:n]


@pytest.mark.parametrize("size", [0, -70, 20])
def test_quotients_closer_to_ties_than_64_bits_tell(size):
    """In whole numbers: the nearest code, where 127 x norm / largest in 64 bits is a tie; and exact ties, to even."""
    top_norm, found = next_to_ties(300, 4)
    rows, cols = len(found), -(-(len(found) + 2) // 16) * 16
    x, norm, want = np.zeros((rows, cols), np.float32), np.ones(cols, np.float32), np.zeros((rows, cols), np.int8)
    norm[0], want[:, 0], odd = top_norm, 127, 0
    for i, (a, b, top, k, off) in enumerate(found):
        sign = -1 if i % 2 else 1
        x[i, 0], x[i, 1 + i], norm[1 + i], want[i, 1 + i] = top, sign * a, b, sign * (k + (off > 0))
        odd += int(np.rint(a * b * 127.0 / (top * top_norm))) != k + (off > 0)
    assert odd > 3  # some of them are what they are for
    x[5, :], want[5, :] = 0, 0
    x[5, 0], x[5, -1], want[5, 0], want[5, -1] = 254, 3, 127, 0
    norm[-1] = top_norm  # 254 and 3: 1.5, to 2
    want[5, -1] = 2
    codes, _ = run_quantize((x * 2.0 ** (size - 24)).astype(np.float32), (norm * 2.0 ** -24).astype(np.float32))
    assert np.array_equal(codes, want), np.argwhere(codes != want)[:5]
