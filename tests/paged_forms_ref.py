"""Attention over paged caches with a window and first slots, in float64 numpy: rows of a sequence at once.  (With
shared prefixes the definition is the plain one of paged_ref.py.)"""
import numpy as np
from paged_ref import D


def seen(own, n, window=None, sinks=0):
    """Whether the token at slot `own` (one, or an array as a column) sees slots 0 .. n - 1."""
    p = np.arange(n)
    see = p <= own
    if window is not None:
        see = see & ((own - p < window) | (p < sinks))
    return see


def attention(pool, q, q_lens, kv_lens, tables, window=None, sinks=0, scale=None):
    """(out, bound of |k| . |q| |scale|, largest |v|); pages outside the pool take no part."""
    scale = D ** -0.5 if scale is None else scale
    heads = q.shape[1]
    group = heads // pool.n_kv
    out = np.zeros(q.shape)
    reach, vmax, t = 0.0, 0.0, 0
    for s, (m, n) in enumerate(zip(q_lens, kv_lens)):
        own = (n - m + np.arange(m))[:, None]
        see = seen(own, n, window, sinks)
        p = np.nonzero(see.any(0))[0]
        page = np.asarray(tables[s])[p // pool.page]
        there = (page >= 0) & (page < pool.n_pages)
        p, page = p[there], page[there]
        see = see[:, p]
        k, v = (pool.values(i, page.astype(np.int64) * pool.page + p % pool.page) for i in range(2))
        rows = see.any(1)
        if rows.any():
            vmax = max(vmax, float(np.abs(v).max()))
            for h in range(heads):
                kk, vv, qq = k[:, h // group], v[:, h // group], q[t:t + m, h].astype(np.float64)
                x = np.where(see, qq @ kk.T * scale, -np.inf)[rows]
                w = np.exp(x - x.max(-1, keepdims=True))
                out[t:t + m, h][rows] = w @ vv / w.sum(-1, keepdims=True)
                reach = max(reach, float((np.abs(qq) @ np.abs(kk).T * see).max() * abs(scale)))
        t += m
    return out, reach, vmax
