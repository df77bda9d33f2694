"""How far the attention over paged caches may be from its float64 definition in root mean square.

A rounding to fp16 is off by something within half a step, spread evenly: for values of [2^k, 2^(k+1)) the
half step is 2^(k - 11) and its rms 2^(k - 11) / sqrt 3, so at most 2^-11 / sqrt 3 of the values' rms.  Where
each of a row's probabilities is rounded, the errors of a sum's terms are independent: their rms to that of the
outputs is the same.  n independent roundings: sqrt n times that.

fp16 queries: the probabilities and the outputs are rounded, and in chunks over q8 the products of
probability and V's scale.

fp32 queries: no rounding to fp16.  What is left: a score is 16 sums in fp32 (two parts, 32 or 16 values deep),
off by at most 2^-23 each of the sum's magnitudes, `reach`, and its query parts carry 22 bits; an error e of a
score changes its weight by e.  Numerators and denominators are sums of `steps` products and some joins, at most
2^-23 each; probabilities (22 bits), exponentials, factors and the output's own rounding are 2^-20 together.

A single row may have one weight, and one value of a group, that make up its output.  Roundings are not averaged
then: n of them are off by up to n half steps, n 2^-11 = sqrt(3 n) (sqrt n 2^-11 / sqrt 3), three times the bound
above for n = 3 and 2.45 times for n = 2; the bound for fp32 queries counts largest errors already and holds for a
row too.  Every row has three times the bound."""
import numpy as np

ROUNDING = 2.0 ** -11 / 3 ** 0.5


def chunked(m, group):
    """Whether m new tokens of a sequence take the chunk kernel."""
    return m * group > 16


def rms_bound(fp16, q8, chunk, reach, slots):
    if fp16:
        return ROUNDING * (3 if q8 and chunk else 2) ** 0.5
    return reach * (16 * 2.0 ** -23 + 2.0 ** -22) + (slots / 32 + 64) * 2 * 2.0 ** -23 + 2.0 ** -20


def rms(x, axis=None):
    return np.sqrt((np.asarray(x, np.float64) ** 2).mean(axis))


def check(got, want, bound, floor=0.0):
    """Every row (the last axis) and all of them together; floor: rms that fp16's smallest step allows."""
    err, size = rms(got - want, -1), rms(want, -1)
    assert np.isfinite(err).all()
    over = err - 3 * (bound * size + floor)
    assert (over <= 0).all(), (np.unravel_index(over.argmax(), over.shape), float((err / np.maximum(size, 1e-300)).max()), bound)
    assert rms(got - want) <= bound * rms(want) + floor, (rms(got - want) / rms(want), bound)
