"""The operators on paged caches from their definitions, in float64 numpy, and how far fp32 / fp16
arithmetic may be from them."""
import numpy as np

D, GROUP = 128, 32


def rope_table(rows, rot, base=5000000.0):
    a = np.arange(rows)[:, None] / base ** (np.arange(0, rot, 2) / max(rot, 1))
    return np.stack([np.cos(a), np.sin(a)], axis=-1).astype(np.float32)


def norm_rotate(x, w, cs, rot, interleaved, eps=1e-6):
    """x [T][n][128], cs [T][rot / 2][2]."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    i = np.arange(rot // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    c, s = (cs[:, None, :, k].astype(np.float64) for k in (0, 1))
    a, b = y[..., lo], y[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    return y


def q8_scale(amax):
    """The smallest fp16 that reaches amax / 127."""
    s = (amax / 127).astype(np.float16)
    up = np.nextafter(s, np.float16(np.inf))
    return np.where(s.astype(np.float64) * 127 < amax, up, s)


class Pool:
    """A pool on the host: exact values, and the bytes of its buffers.  Slots that nothing wrote hold NaN
    (fp16 values; the scales of q8)."""

    def __init__(self, fmt, n_kv, page, n_pages):
        self.fmt, self.n_kv, self.page, self.n_pages = fmt, n_kv, page, n_pages
        shape = (n_pages, n_kv, page, D)
        self.q8 = fmt == 1
        self.data = [np.full(shape, 113 if self.q8 else np.nan, np.int8 if self.q8 else np.float16) for _ in "kv"]
        self.scales = [np.full(shape[:3] + (D // GROUP,), np.nan, np.float16) for _ in "kv"]

    def where(self, slots):
        return np.asarray(slots) // self.page, slice(None), np.asarray(slots) % self.page

    def fill(self, slots, rng):
        """Random rows at these pool slots (keys with a few large channels)."""
        n = (len(slots), self.n_kv, D)
        for i in range(2):
            if self.q8:
                self.data[i][self.where(slots)] = rng.integers(-127, 128, n)
                self.scales[i][self.where(slots)] = rng.uniform(0.002, 0.03, n[:2] + (D // GROUP,))
            else:
                x = rng.standard_normal(n)
                if i == 0:
                    x[..., 5::37] *= 4
                self.data[i][self.where(slots)] = x

    def values(self, i, slots):
        """[len(slots)][n_kv][128] float64."""
        x = self.data[i][self.where(slots)].astype(np.float64)
        if not self.q8:
            return x
        return x * np.repeat(self.scales[i][self.where(slots)].astype(np.float64), GROUP, axis=-1)


def attention(pool, q, q_lens, kv_lens, tables, scale=None):
    """(out, bound of |k| . |q| |scale|, largest |v|); q [T][heads][128], pages outside the pool take no part."""
    scale = D ** -0.5 if scale is None else scale
    heads = q.shape[1]
    group = heads // pool.n_kv
    out = np.zeros(q.shape)
    reach, vmax, t = 0.0, 0.0, 0
    for s, (m, n) in enumerate(zip(q_lens, kv_lens)):
        p = np.arange(n)
        page = np.asarray(tables[s])[p // pool.page] if n else p
        there = (page >= 0) & (page < pool.n_pages)
        slots = np.where(there, page, 0) * pool.page + p % pool.page
        k, v = pool.values(0, slots), pool.values(1, slots)
        for i in range(m):
            see = there & (p <= n - m + i)
            if not see.any():
                continue
            for h in range(heads):
                kk, vv, qq = k[see, h // group], v[see, h // group], q[t + i, h].astype(np.float64)
                x = kk @ qq * scale
                w = np.exp(x - x.max())
                out[t + i, h] = w @ vv / w.sum()
                reach = max(reach, float((np.abs(kk) @ np.abs(qq)).max() * abs(scale)))  # a scale may be negative
                vmax = max(vmax, float(np.abs(vv).max()))
        t += m
    return out, reach, vmax


def attention_tol(fp16, q8, reach, vmax):
    """How far an output may be from the exact one.  fp32: a score is a sum of 128 products whose
    operands carry 22 bits (2^-21 for the two of them), accumulated in fp32 (at most 128 roundings,
    2^-17): reach (2^-21 + 2^-17); a score error e changes every weight by a factor within e^(+-e) and so
    the output by at most 2 e vmax; probabilities carry 22 bits and their sums are fp32.  fp16: the
    probabilities are rounded to fp16 (2^-11 of the output's terms), the output too, and for q8 the
    dequantised keys (2^-11 of a score's products) and values."""
    e = reach * (2.0 ** -21 + 2.0 ** -17)
    tol = 2.0 ** -18
    if fp16:
        tol += (3 if q8 else 2) * 2.0 ** -11
        e += reach * 2.0 ** -11 if q8 else 0.0
    return (2 * e + tol) * vmax
