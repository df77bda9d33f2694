"""CPU tests of the bounds in paged_bounds.py: arithmetic that loses what the kernels keep (keys rounded to
fp16, the low part of a query, a probability or a value, a slot too few or too many) is outside, the kernels'
own roundings are inside.  The mistakes are made in the definition, in numpy."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import paged_bounds as bounds  # noqa: E402
import paged_ref as ref  # noqa: E402

D = ref.D


def half(x):
    return x.astype(np.float16).astype(np.float64)


def inputs(q8, spread, slots=600, rows=24, seed=1):
    """q, k, v of one head; scores of about `spread` in rms."""
    rng = np.random.default_rng(seed)
    pool = ref.Pool(1 if q8 else 0, 1, slots, 1)
    pool.fill(np.arange(slots), rng)
    k, v = (pool.values(i, np.arange(slots))[:, 0] for i in range(2))
    q = rng.standard_normal((rows, D))
    return q * spread / bounds.rms(q @ k.T * D ** -0.5), k, v


def attend(q, k, v, p_of=lambda p: p, denominator_of=None, vs=None):
    s = q @ k.T * D ** -0.5
    p = np.exp(s - s.max(-1, keepdims=True))
    w = p_of(p)
    d = (denominator_of or p_of)(p)
    if vs is None:
        return w @ v / d.sum(-1, keepdims=True)
    codes = v / np.where(vs > 0, vs, 1)
    out = [half(w * vs[:, g * 32][None]) @ codes[:, g * 32:g * 32 + 32] for g in range(4)]
    return np.concatenate(out, -1) / d.sum(-1, keepdims=True)


def bound_of(fp16, q8, chunk, q, k):
    return bounds.rms_bound(fp16, q8, chunk, float((np.abs(q) @ np.abs(k).T).max() * D ** -0.5), len(k))


def outside(got, want, bound):
    with pytest.raises(AssertionError):
        bounds.check(got, want, bound)


@pytest.mark.parametrize("spread", [0.05, 1.0, 4.0])
@pytest.mark.parametrize("q8", [False, True])
def test_the_kernels_roundings_are_inside(q8, spread):
    q, k, v = inputs(q8, spread)
    q = half(q)
    want = attend(q, k, v)
    bounds.check(half(attend(q, k, v, half)), want, bound_of(True, q8, False, q, k))
    bounds.check(half(attend(q, k, v, half, lambda p: p)), want, bound_of(True, q8, False, q, k))
    if q8:
        scale = np.repeat(np.abs(v).reshape(-1, 4, 32).max(-1) / 127, 32, -1).astype(np.float16).astype(np.float64)
        v = np.rint(v / scale) * scale
        want = attend(q, k, v)
        bounds.check(half(attend(q, k, v, half, vs=scale)), want, bound_of(True, True, True, q, k))
    bounds.check(attend(q.astype(np.float32).astype(np.float64), k, v).astype(np.float32), want, bound_of(False, q8, True, q, k))


def test_keys_rounded_to_fp16_are_outside():
    q, k, v = inputs(True, 4.0)
    q = half(q)
    for chunk in (False, True):
        outside(half(attend(q, half(k), v, half)), attend(q, k, v), bound_of(True, True, chunk, q, k))
    outside(attend(q, half(k), v), attend(q, k, v), bound_of(False, True, True, q, k))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("spread", [1.0, 4.0])
def test_a_lost_low_part_is_outside_for_fp32_queries(q8, spread):
    q, k, v = inputs(q8, spread)
    want, bound = attend(q, k, v), bound_of(False, q8, True, q, k)
    outside(attend(half(q), k, v), want, bound)
    if spread > 1:  # few large weights: their own errors cancel against the denominator's, and reach is large
        return
    outside(attend(q, k, v, half, lambda p: p), want, bound)
    if q8:
        outside(attend(q, k, half(v)), want, bound)


@pytest.mark.parametrize("fp16", [False, True])
def test_a_slot_too_few_or_too_many_is_outside(fp16):
    q, k, v = inputs(True, 1.0)
    q = half(q) if fp16 else q
    want = attend(q[:, :], k[:-1], v[:-1])
    outside(attend(q, k, v), want, bound_of(fp16, True, True, q, k))
    outside(attend(q, k[:-2], v[:-2]), want, bound_of(fp16, True, True, q, k))
    v2 = v[:-1].copy()
    v2[100, 32:64] *= 2  # one scale of one slot
    outside(attend(q, k[:-1], v2), want, bound_of(fp16, True, True, q, k))
