"""Operators of a layer that serves a batch of sessions, timed against their plain forms.

``project`` and ``gated`` are the layer's matrix products on 8-bit integers: the tokens' rows are (normalised and)
quantised with one scale a token, multiplied by a matrix with one scale an output channel, and end as rows of y,
with a residual added (project), or as silu(gate) * up of two matrices (gated).  ``window`` and ``prefix`` are two
forms of attention over paged K/V caches: over a window of the last slots and a few first ones that stay visible,
and for sessions that share a long prefix, whose slots are read once for all of them.

``listed`` names the cases, ``draw`` gives more of the same ranges, ``prepare`` makes what a program has in hand
before the call, ``run`` is one pass (with ``own`` through the library, else in elementary torch operations),
``work`` the bytes and operations a pass cannot do without and ``exact`` the same outputs from the definitions in
64-bit arithmetic.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

D = 128     # head dimension
GROUP = 32  # values that share a q8 scale
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}


def listed():
    return [
        # The q|k|v rows of one decode step of eight sessions: the smallest call, latency.
        {"name": "project_8_qkv", "kind": "project", "rows": 8, "k": 2048, "n": 4096, "x": "f32", "y": "f32",
         "norm": True, "add": False},
        # The logits of 64 sessions: the largest matrix, read once.
        {"name": "project_64_logits", "kind": "project", "rows": 64, "k": 2048, "n": 151936, "x": "f32", "y": "f16",
         "norm": True, "add": False},
        # The attention's output product behind four follow-up turns of 41 tokens, added to the residual.
        {"name": "project_164_o", "kind": "project", "rows": 164, "k": 2048, "n": 2048, "x": "f16", "y": "f32",
         "norm": False, "add": True},
        # The feed-forward block's second product for a whole prompt, added to the residual.
        {"name": "project_4096_down", "kind": "project", "rows": 4096, "k": 6144, "n": 2048, "x": "f16", "y": "f32",
         "norm": False, "add": True},
        # The feed-forward block's first products for sixteen sessions' tokens.
        {"name": "gated_16", "kind": "gated", "rows": 16, "k": 2048, "n": 6144, "x": "f32", "y": "f16", "norm": True},
        # The same for a whole prompt: the most operations.
        {"name": "gated_4096", "kind": "gated", "rows": 4096, "k": 2048, "n": 6144, "x": "f32", "y": "f16", "norm": True},
        # A step of 32 long sessions, of which each sees its last 1024 slots and four first ones.
        {"name": "window_decode_32", "kind": "window", "fmt": "f16", "type": "f32", "seqs": 32, "ctx": 16384, "q": 1,
         "heads": 16, "kv": 8, "page": 64, "mixed": False, "window": 1024, "sinks": 4},
        # A whole prompt through a window of an eighth of it.
        {"name": "window_prompt_4096", "kind": "window", "fmt": "f16", "type": "f16", "seqs": 1, "ctx": 4096, "q": 4096,
         "heads": 16, "kv": 8, "page": 64, "mixed": False, "window": 512, "sinks": 16},
        # Chunks of prompts and single tokens of sessions over quantised caches.
        {"name": "window_mixed_q8", "kind": "window", "fmt": "q8", "type": "f16", "seqs": 12, "ctx": 8192, "q": 500,
         "heads": 16, "kv": 8, "page": 32, "mixed": True, "window": 2048, "sinks": 64},
        # A step of 64 sessions behind one system prompt and screenshot.
        {"name": "prefix_decode_64", "kind": "prefix", "fmt": "f16", "type": "f16", "seqs": 64, "ctx": 8192, "q": 1,
         "heads": 16, "kv": 8, "page": 64, "mixed": False, "groups": 1, "prefix": 7680, "alone": 0},
        # Eight drafts each of sessions of three kinds, some of which share nothing, over quantised caches.
        {"name": "prefix_drafts_q8", "kind": "prefix", "fmt": "q8", "type": "f32", "seqs": 20, "ctx": 4096, "q": 8,
         "heads": 16, "kv": 8, "page": 32, "mixed": False, "groups": 3, "prefix": 2976, "alone": 2},
        # Follow-up turns of sessions behind one prefix, beside single tokens.
        {"name": "prefix_chunks_16", "kind": "prefix", "fmt": "f16", "type": "f16", "seqs": 16, "ctx": 6000, "q": 200,
         "heads": 16, "kv": 8, "page": 16, "mixed": True, "groups": 1, "prefix": 5008, "alone": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(16, 8), (16, 8), (16, 8), (4, 4), (12, 4), (10, 2), (16, 1), (24, 8)]
PAGES = [16, 32, 48, 64, 64, 128, 256]


def draw(rng):
    kind = rng.choice(["project", "gated", "window", "window", "prefix", "prefix"])
    types = ["f32", "f16"]
    if kind in ("project", "gated"):
        rows = _log_int(rng, 1, 4096)
        k = 16 * _log_int(rng, 8, 512)
        n = _log_int(rng, 24, min(16384, max(24, 4096 * 6144 * 2048 // (rows * k))))
        case = {"kind": kind, "rows": rows, "k": k, "n": n, "x": rng.choice(types), "y": rng.choice(types),
                "norm": rng.random() < 0.5}
        return case | {"add": rng.random() < 0.5} if kind == "project" else case
    heads, kv = rng.choice(HEADS)
    fmt, page, type_ = rng.choice(["f16", "q8"]), rng.choice(PAGES), rng.choice(types)
    shape = rng.choice(["decode", "decode", "drafts", "chunk", "mixed"])
    if shape in ("decode", "drafts"):
        seqs = _log_int(rng, 1 if kind == "window" else 2, 64)
        ctx = _log_int(rng, 64, min(16384, 150000 // seqs))
        q = 1 if shape == "decode" else rng.randint(2, 12)
    else:
        seqs, heads = _log_int(rng, 1 if kind == "window" else 2, 12), min(heads, 2 * kv)
        ctx = _log_int(rng, 128, int(8192 / math.sqrt(seqs)))
        q = _log_int(rng, 13, max(13, min(ctx // 2, 4096 // seqs)))
    case = {"kind": kind, "fmt": fmt, "type": type_, "seqs": seqs, "ctx": ctx, "q": q, "heads": heads, "kv": kv, "page": page,
            "mixed": shape == "mixed"}
    if kind == "window":
        return case | {"window": _log_int(rng, 16, 4096), "sinks": rng.choice([0, 1, 4, 16, 64, 200])}
    groups = min(rng.choice([1, 1, 2, 4]), seqs)
    return case | {"groups": groups, "prefix": _log_int(rng, max(8, (ctx - q) // 16), max(8, ctx - q)) // page * page,
                   "alone": rng.choice([0, 0, 1]) if seqs > groups else 0}


# ---------------------------------------------------------------------------------------------
# What a program has in hand

def _lengths(case):
    """(slots in use, new tokens) of every sequence: the first has the case's, the others anything from an eighth of
    the slots (prefix: of those behind it); in a mixed batch every other sequence decodes a single token."""
    r = random.Random(case["seqs"] * 1000003 + case["ctx"] * 101 + case["q"])
    least = case.get("prefix", 0)
    kv, q = [case["ctx"]], [case["q"]]
    for i in range(1, case["seqs"]):
        m = case["q"]
        if case["mixed"]:
            m = 1 if i % 2 else _log_int(r, max(1, m // 4), m)
        behind = case["ctx"] - least
        kv.append(least + _log_int(r, min(behind, max(m, behind // 8)), behind))
        q.append(m)
    return kv, q


def _groups(case):
    """First sequence of every group, and one more: the end of the last; those behind it share nothing."""
    n = case["seqs"] - case["alone"]
    return [n * g // case["groups"] for g in range(case["groups"] + 1)]


def _prefixes(case):
    """Shared slots of every group, whole pages: the first has the case's."""
    return [max(0, (case["prefix"] // case["page"] - 3 * g) * case["page"]) for g in range(case["groups"])]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, *shape):
    """Rows as a decoder has them: a few channels much larger than the others."""
    x = torch.randn(*shape, device="cuda", generator=g)
    x[..., 5::37] *= 4
    return x


def _pool(case, g, pages):
    """A pool whose pages have all been written before: (k, v, scales of k, of v)."""
    shape = (pages, case["kv"], case["page"], D)
    if case["fmt"] == "f16":
        return [_activations(g, *shape).half(), torch.randn(*shape, device="cuda", generator=g).half(), None, None]
    codes = [torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [(torch.rand(*shape[:3], D // GROUP, device="cuda", generator=g) * 0.03 + 0.002).half() for _ in range(2)]
    return codes + scales


def _tables(case, kv, seed):
    """Page tables over shuffled pages: (table, pages of the pool).  A group's sequences have the pages of its prefix
    in common; pages in front of a window that no token sees any more have been given back (-1)."""
    page = case["page"]
    need = [-(-n // page) for n in kv]
    shared = [0] * len(kv)  # pages of the sequence that are its group's
    leader = list(range(len(kv)))
    if case["kind"] == "prefix":
        starts = _groups(case)
        for g, n in enumerate(_prefixes(case)):
            for s in range(starts[g], starts[g + 1]):
                shared[s], leader[s] = n // page, starts[g]
    pages = sum(n - (c if l != s else 0) for s, (n, c, l) in enumerate(zip(need, shared, leader))) + 3
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table, at = np.zeros((len(kv), max(need)), dtype=np.int32), 0
    for s, n in enumerate(need):
        c = shared[s] if leader[s] != s else 0
        table[s, :c] = table[leader[s], :c]
        table[s, c:n] = order[at:at + n - c]
        at += n - c
    if case["kind"] == "window":
        for s, (n, m) in enumerate(zip(kv, _lengths(case)[1])):
            first = -(-case["sinks"] // page)
            last = max(0, n - m + 1 - case["window"]) // page
            table[s, first:max(first, last)] = -1
    return table, pages


class OnDevice:
    """A torch tensor as the library takes device memory: by its address."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.nbytes


def _prepare_product(case, s, g):
    rows, k = case["rows"], case["k"]
    n = case["n"] * (2 if case["kind"] == "gated" else 1)
    s["x"] = _activations(g, rows, k).mul_(1.5).to(TYPES[case["x"]])
    s["norm"] = 1 + 0.3 * torch.randn(k, device="cuda", generator=g) if case["norm"] else None
    # A matrix as it is kept: rounded to 8 bits, each output channel by its own largest value.
    s["w"] = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8)
    s["w_scales"] = (torch.rand(n, device="cuda", generator=g) * 0.8 + 0.6) * (0.02 / 74 * math.sqrt(2048 / k))
    s["add"] = torch.randn(rows, case["n"], device="cuda", generator=g) if case.get("add") else None
    s["y"] = torch.empty(rows, case["n"], device="cuda", dtype=TYPES[case["y"]])
    if own:
        from instantcua_amd import engine as eng
        from instantcua_amd import int8
        s["codes"] = eng.DeviceBuffer(rows * k)
        s["scales"] = eng.DeviceBuffer(4 * rows)
        need = int8.matmul_work(rows, case["n"], k, gated=case["kind"] == "gated")
        s["work"] = eng.DeviceBuffer(need) if need else None
    return s


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["kind"] in ("project", "gated"):
        _prepare_product(case, s, g)
    else:
        kv, q = _lengths(case)
        table, pages = _tables(case, kv, seed)
        s["pool"] = _pool(case, g, pages)
        s["tables"] = torch.from_numpy(table).cuda()
        s["kv_len"] = torch.tensor(kv, device="cuda", dtype=torch.int32)
        s["q_start"] = torch.tensor([0] + list(np.cumsum(q)), device="cuda", dtype=torch.int32)
        s["n"], s["max_q"], s["max_kv"] = sum(q), max(q), max(kv)
        if case["kind"] == "prefix":
            s["group_start"] = torch.tensor(_groups(case), device="cuda", dtype=torch.int32)
            s["prefix_len"] = torch.tensor(_prefixes(case), device="cuda", dtype=torch.int32)
            s["max_prefix"] = max(_prefixes(case))
        s["q"] = (torch.randn(s["n"], case["heads"], D, device="cuda", generator=g) * 1.3).to(TYPES[case["type"]])
        s["out"] = torch.empty_like(s["q"])
        if own:  # the handle that a program keeps for its cache, and the attention's workspace
            from instantcua_amd import engine as eng
            from instantcua_amd import paged
            from instantcua_amd.modelfile import WeightFormat
            buffers = [None if t is None else OnDevice(t) for t in s["pool"]]
            s["cache"] = paged.PagedCache(WeightFormat.Q8 if case["fmt"] == "q8" else WeightFormat.F16, case["kv"],
                                          case["page"], s["pool"][0].shape[0], *buffers)
            sizes = {"max_q": s["max_q"], "max_kv": s["max_kv"]}
            if case["kind"] == "window":
                need = s["cache"].attention_window_work(case["heads"], len(kv), s["n"], case["window"], case["sinks"], **sizes)
            else:
                need = s["cache"].attention_prefix_work(case["heads"], len(kv), s["n"], case["groups"], s["max_prefix"], **sizes)
            s["work"] = eng.DeviceBuffer(need) if need else None
    if own:
        s["dev"] = {k: OnDevice(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
    return s


# ---------------------------------------------------------------------------------------------
# One pass

def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


def _run_own(s):
    from instantcua_amd import int8, paged
    case, d = s["case"], s["dev"]
    stream = torch.cuda.current_stream().cuda_stream
    types = {"f32": paged.F32, "f16": paged.F16}
    if case["kind"] in ("project", "gated"):
        int8.quantize(d["x"], s["codes"], s["scales"], case["rows"], case["k"], norm=d.get("norm"), eps=EPS,
                      type=types[case["x"]], stream=stream)
        int8.matmul(s["codes"], s["scales"], d["w"], d["w_scales"], d["y"], case["rows"], case["n"], case["k"],
                    add=d.get("add"), gated=case["kind"] == "gated", type=types[case["y"]], work=s["work"], stream=stream)
        return s["y"]
    rest = {"max_q": s["max_q"], "max_kv": s["max_kv"], "type": types[case["type"]], "work": s["work"], "stream": stream}
    sizes = (len(s["kv_len"]), s["n"], s["tables"].shape[1])
    if case["kind"] == "window":
        s["cache"].attention_window(d["q"], d["out"], case["heads"], d["q_start"], d["kv_len"], d["tables"], *sizes,
                                    case["window"], case["sinks"], **rest)
    else:
        s["cache"].attention_prefix(d["q"], d["out"], case["heads"], d["q_start"], d["kv_len"], d["tables"], *sizes,
                                    d["group_start"], d["prefix_len"], case["groups"], s["max_prefix"], **rest)
    return s["out"]


def _quantise(s):
    """Codes (as fp32) and scales of the rows.  The root mean square is common to a row's values, so codes are of the
    values before it; in 64 bits, as a value next to the border of two codes has to fall to the right one."""
    x = s["x"].float()
    t = x.double()
    scale = torch.ones(x.shape[0], 1, device="cuda")
    if s["norm"] is not None:
        t = t * s["norm"].double()
        scale = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    top = t.abs().amax(-1, keepdim=True)
    codes = torch.round(t * 127 / torch.where(top > 0, top, torch.ones_like(top)))
    return codes.float(), top.float() * scale / 127


def _product(codes, w):
    """Sums of products of codes over parts of K whose every partial sum is below 2^24: exact in fp32; the parts are
    added in 64 bits."""
    out = torch.zeros(codes.shape[0], w.shape[0], device="cuda", dtype=torch.float64)
    for k in range(0, w.shape[1], 1024):
        out += codes[:, k:k + 1024] @ w[:, k:k + 1024].float().t()
    return out.float()


def _project(s):
    codes, scales = _quantise(s)
    y = _product(codes, s["w"]) * scales * s["w_scales"]
    if s["add"] is not None:
        y = y + s["add"]
    return y.to(s["y"].dtype)


def _gated(s):
    codes, scales = _quantise(s)
    n = s["case"]["n"]
    gate, up = ((_product(codes, s["w"][i:i + n]) * scales * s["w_scales"][i:i + n]) for i in (0, n))
    return (gate / (1 + torch.exp(-gate)) * up).to(s["y"].dtype)


def _values(pool, i, pages, slots):
    """fp32 values of k (i = 0) or v (i = 1) at (page, slot): [..., kv, D]."""
    x = pool[i][pages, :, slots].float()
    if pool[2 + i] is not None:
        sc = pool[2 + i][pages, :, slots].float()
        x = (x.unflatten(-1, (D // GROUP, GROUP)) * sc.unsqueeze(-1)).flatten(-2)
    return x


def _attention(s):
    """Sequences padded to the longest, some at a time: scores, the softmax's exponentials and their sum, and the
    weighted values, all in 32 bits."""
    case = s["case"]
    S, Q, L, n = len(s["kv_len"]), s["max_q"], s["max_kv"], case["kv"]
    G = case["heads"] // n
    at, rows = torch.arange(L, device="cuda"), torch.arange(Q, device="cuda")
    out = torch.empty(s["n"], case["heads"], D, device="cuda", dtype=s["q"].dtype)
    part = max(1, 2 ** 30 // (n * L * max(2 * D, Q * G)))
    for s0 in range(0, S, part):
        table, kv_len = s["tables"][s0:s0 + part].long(), s["kv_len"][s0:s0 + part].long()
        B = len(kv_len)
        start, end = s["q_start"][s0:s0 + B].long(), s["q_start"][1 + s0:1 + s0 + B].long()
        page = table[:, at // case["page"]]
        slot = (at % case["page"]).expand(B, L)
        k, v = (_values(s["pool"], i, page.clamp(min=0), slot).transpose(1, 2).reshape(B * n, L, D) for i in range(2))
        valid = rows < (end - start)[:, None]
        index = (start[:, None] + rows).clamp(max=s["n"] - 1)
        q = s["q"].float()[index].view(B, Q, n, G, D).permute(0, 2, 1, 3, 4).reshape(B * n, Q * G, D)
        score = torch.bmm(q, k.transpose(1, 2)) * (1 / math.sqrt(D))
        last = (kv_len - (end - start))[:, None] + rows  # the row's own slot
        last = torch.where(valid, last, last.new_full((), L - 1))[..., None]
        seen = at <= last
        if case["kind"] == "window":
            seen = seen & ((at > last - case["window"]) | (at < case["sinks"]))
        seen = seen[:, None, :, None].expand(B, n, Q, G, L).reshape(B * n, Q * G, L)
        score = score.masked_fill_(~seen, -math.inf)
        score = score.sub_(score.amax(-1, keepdim=True)).exp_()
        y = torch.bmm(score, v) / score.sum(-1, keepdim=True)
        y = y.view(B, n, Q, G, D).permute(0, 2, 1, 3, 4).reshape(B, Q, case["heads"], D)
        out[index[valid]] = y[valid].to(out.dtype)
    return out


_PLAIN = {"project": _project, "gated": _gated, "window": _attention, "prefix": _attention}


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without

def _row_bytes(case):
    """Bytes of a key or value of one head."""
    return 2 * D if case["fmt"] == "f16" else D + 2 * D // GROUP


def work(case):
    if case["kind"] in ("project", "gated"):
        rows, k, n = case["rows"], case["k"], case["n"]
        channels = n * (2 if case["kind"] == "gated" else 1)
        b = rows * k * SIZE[case["x"]] + channels * (k + 4) + rows * n * SIZE[case["y"]] + (4 * k if case["norm"] else 0)
        return {"bytes": b + (4 * rows * n if case.get("add") else 0), "flops": 2 * rows * k * channels}
    kv, q = _lengths(case)
    pairs, slots = 0, 0
    for c, m in zip(kv, q):
        if case["kind"] == "window":
            p = np.arange(c - m, c)
            first = np.maximum(0, p - case["window"] + 1)
            pairs += int(np.sum(p + 1 - first + np.minimum(first, case["sinks"])))
            slots += int(c - first[0] + min(first[0], case["sinks"]))
        else:
            pairs += m * (c - m) + m * (m + 1) // 2
            slots += c
    if case["kind"] == "prefix":
        starts = _groups(case)
        slots -= sum(p * (max(1, starts[g + 1] - starts[g]) - 1) for g, p in enumerate(_prefixes(case)))
    return {"bytes": 2 * slots * case["kv"] * _row_bytes(case) + 2 * sum(q) * case["heads"] * D * SIZE[case["type"]],
            "flops": 4 * D * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------
# The same in 64 bits

def _exact_product(case, s):
    x, rows, n = s["x"].double(), case["rows"], case["n"]
    codes, scale = torch.empty(rows, case["k"], dtype=torch.float64, device="cuda"), torch.empty(rows, 1, dtype=torch.float64, device="cuda")
    for r in range(0, rows, 512):
        y = x[r:r + 512]
        if s["norm"] is not None:
            y = y * s["norm"].double()
        largest = torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True)
        codes[r:r + 512] = torch.round((y * 127) / largest)
        scale[r:r + 512] = largest / 127
        if s["norm"] is not None:
            scale[r:r + 512] /= (torch.linalg.vector_norm(x[r:r + 512], dim=-1, keepdim=True) ** 2 / case["k"] + EPS).sqrt()
    y = torch.empty(rows, s["w"].shape[0], dtype=torch.float64, device="cuda")
    for c in range(0, s["w"].shape[0], 8192):
        w = s["w"][c:c + 8192].double() * s["w_scales"][c:c + 8192].double()[:, None]
        y[:, c:c + 8192] = torch.mm(codes * scale, w.t())
    if case["kind"] == "gated":
        return y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
    return y if s["add"] is None else y + s["add"].double()


def _exact_rows(s, i, slots, page):
    """Values at pool slots, [n, kv, D]."""
    x = s["pool"][i][slots // page, :, slots % page].double()
    if s["pool"][2 + i] is None:
        return x
    return x * s["pool"][2 + i][slots // page, :, slots % page].double().repeat_interleave(GROUP, dim=-1)


@torch.no_grad()
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["kind"] in ("project", "gated"):
        return _exact_product(case, s)
    kv, q = _lengths(case)
    G = case["heads"] // case["kv"]
    out, at = torch.empty(sum(q), case["heads"], D, dtype=torch.float64, device="cuda"), 0
    for i, (c, m) in enumerate(zip(kv, q)):
        # The slots that some token of the sequence sees, then, token by token, which of them.
        p = torch.arange(c, device="cuda")
        if case["kind"] == "window":
            p = p[(p < case["sinks"]) | (p >= c - m + 1 - case["window"])]
        slots = s["tables"][i].long()[p // case["page"]] * case["page"] + p % case["page"]
        K, V = (_exact_rows(s, j, slots, case["page"]) for j in range(2))
        for h in range(case["heads"]):
            kh, vh = K[:, h // G].contiguous(), V[:, h // G].contiguous()
            for r in range(0, m, 1024):
                x = s["q"][at + r:at + min(m, r + 1024), h].double()
                w = x @ kh.t() / math.sqrt(D)
                own_slot = (c - m + r + torch.arange(len(x), device="cuda"))[:, None]
                hidden = p > own_slot
                if case["kind"] == "window":
                    hidden |= (own_slot - p >= case["window"]) & (p >= case["sinks"])
                out[at + r:at + r + len(x), h] = torch.softmax(w.masked_fill_(hidden, -math.inf), -1) @ vh
        at += m
    return out
