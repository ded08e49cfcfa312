"""Serving operators: a paged 8-bit KV cache, the attention that reads it, and
the choice of the next token.

A program that serves many requests at once with this framework keeps the keys
and values of all of them in one pool of pages.  Each step it works out which
pages and which slots the new tokens take (``page_plan``), writes their keys and
values there in 8 bits (``kv_store_paged``), attends over what the pool holds
(``attention_paged``), and draws each request's next token from the logits
(``sample``).

Layouts.  A page holds P tokens of every key/value head: ``k_cache``
[pages, Hkv, P, hd] and ``v_cache`` [pages, Hkv, hd, P] in e4m3, ``k_scale`` and
``v_scale`` [pages, Hkv] in float32, one scale per page and head.  The scales
that ``kv_store_paged`` writes are powers of two.  A slot is page * P + place.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # the bookkeeping of one decode step: one new token per request
        {"name": "plan_decode", "op": "plan", "batch": 64, "new": 1, "len": 4096, "page": 64, "spread": 1},
        # a long prompt queue admitted at once, small pages
        {"name": "plan_prompts", "op": "plan", "batch": 500, "new": 2000, "len": 700, "page": 16, "spread": 2},
        # a decode step's keys and values, one token per request
        {"name": "store_decode", "op": "store", "dtype": "bfloat16", "batch": 64, "new": 1, "len": 4096, "page": 64,
         "kv": 8, "hd": 128, "spread": 3},
        # prompts of uneven lengths written at once, some behind a cached prefix
        {"name": "store_prompts", "op": "store", "dtype": "bfloat16", "batch": 12, "new": 2500, "len": 300, "page": 64,
         "kv": 8, "hd": 128, "spread": 4},
        # one user's next token on the repository's decoder (12 heads of 64): latency
        {"name": "attend_one", "op": "attend", "dtype": "bfloat16", "batch": 1, "new": 1, "len": 1000, "page": 16,
         "heads": 12, "kv": 12, "hd": 64, "window": 0, "spread": 5},
        # a decode step of many requests of very uneven lengths, grouped heads
        {"name": "attend_batch", "op": "attend", "dtype": "bfloat16", "batch": 64, "new": 1, "len": 8192, "page": 64,
         "heads": 32, "kv": 8, "hd": 128, "window": 0, "spread": 6},
        # two long documents, one token each: the cache's bytes and nothing else
        {"name": "attend_long", "op": "attend", "dtype": "float16", "batch": 2, "new": 1, "len": 131072, "page": 128,
         "heads": 64, "kv": 8, "hd": 128, "window": 0, "spread": 7},
        # single precision decode over a sliding window
        {"name": "attend_f32", "op": "attend", "dtype": "float32", "batch": 24, "new": 1, "len": 3000, "page": 32,
         "heads": 12, "kv": 12, "hd": 64, "window": 1000, "spread": 8},
        # chunks of long prompts on top of what is cached: the matrix work
        {"name": "attend_prompt", "op": "attend", "dtype": "bfloat16", "batch": 6, "new": 2000, "len": 6000, "page": 64,
         "heads": 32, "kv": 8, "hd": 128, "window": 0, "spread": 9},
        # a chat turn's first pass on the repository's decoder: short ragged prompts
        {"name": "attend_chat", "op": "attend", "dtype": "float16", "batch": 16, "new": 237, "len": 0, "page": 16,
         "heads": 12, "kv": 12, "hd": 64, "window": 0, "spread": 10},
        # the repository's decoder, four users, nucleus sampling: latency
        {"name": "sample_chat", "op": "sample", "dtype": "bfloat16", "batch": 4, "vocab": 32000, "mixed": False},
        # a full serving batch over a large vocabulary, each request with settings of its own
        {"name": "sample_serve", "op": "sample", "dtype": "float32", "batch": 200, "vocab": 131072, "mixed": True},
    ]


def draw(rng):
    """One more case of the same ranges; never more work than the largest listed one."""
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["plan", "store", "store", "attend", "attend", "attend", "attend", "sample", "sample"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "sample":
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, 256), "vocab": _log(rng, 40, 200000),
                "mixed": rng.random() < 0.5}
    c = {"op": op, "dtype": dtype, "batch": _log(rng, 1, 256), "page": rng.choice([16, 32, 64, 64, 128, 256]),
         "spread": rng.randrange(1000)}
    if op == "plan":
        del c["dtype"]
        c.update(batch=_log(rng, 1, 2000), new=rng.choice([1, 1, _log(rng, 1, 3000)]), len=_log(rng, 1, 20000))
        return c
    group, kv, hd = rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 8, 12]), rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    if op == "store":
        c.update(new=rng.choice([1, 1, _log(rng, 1, 4000)]), len=_log(rng, 1, 4000), kv=kv, hd=hd)
        return c
    new = rng.choice([1, 1, rng.randint(2, 5), _log(rng, 8, 2000)])
    c.update(new=new, len=_log(rng, 1, 60000 if new == 1 else 8000), heads=group * kv, kv=kv, hd=hd,
             window=rng.choice([0, 0, 0, _log(rng, 16, 4000)]))
    return c


def _cost(case):
    """Work of a case in the plain form's terms, to keep draws below the listed ones."""
    w = work(case)
    padded = 0.0
    if case["op"] == "attend":
        # the plain form's padded scores and dequantised pages
        lens, new = _lengths(case)
        longest, most = max(lens) + 0.0, max(new)
        padded = case["batch"] * (case["heads"] * most * longest + 2 * case["kv"] * longest * case["hd"]) / 50.0
    elif case["op"] == "store":
        padded = _n_pages(case) * case["page"] * case["kv"] * case["hd"] * 4.0 / 50.0
    return w["bytes"] + w["flops"] / 400.0 + padded


# ---- what a case holds -------------------------------------------------------

def _lengths(case):
    """(tokens each request has in the cache after the step, how many of them are new).

    Spread over the whole range below the case's figures; the first request is
    the longest and the last one, where there are more than two, is short.
    """
    rng = random.Random(case["spread"])
    total, new = [], []
    for i in range(case["batch"]):
        n = case["new"] if case["new"] == 1 or i == 0 else max(1, int(case["new"] * rng.uniform(0.1, 1.0)))
        old = case["len"] - (1 if case["op"] == "attend" and case["new"] == 1 and case["len"] else 0) if i == 0 else int(case["len"] * rng.random())
        if case["batch"] > 2 and i == case["batch"] - 1:
            old = min(old, 3)
        total.append(old + n)
        new.append(n)
    return total, new


def _n_pages(case):
    total, _ = _lengths(case)
    return sum(-(-t // case["page"]) for t in total) + 3


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * SIZE[case["dtype"]] + case["batch"] * 28, "flops": 4.0 * n}
    total, new = _lengths(case)
    P = case["page"]
    if op == "plan":
        taken = sum(-(-t // P) - -(-(t - n) // P) for t, n in zip(total, new))
        return {"bytes": 16 * case["batch"] + 8 * taken + 8 * sum(new), "flops": 0.0}
    row = case["kv"] * case["hd"]
    if op == "store":
        return {"bytes": sum(new) * (2 * row * (SIZE[case["dtype"]] + 1) + 4), "flops": 4.0 * sum(new) * row}
    window = case["window"]
    seen = pairs = 0
    for t, n in zip(total, new):
        # keys that some query of the request sees, and (query, key) pairs
        seen += t if not window else min(t, window + n - 1)
        if not window:
            pairs += n * (t - n) + n * (n + 1) // 2
        else:
            pairs += sum(min(window, t - n + i + 1) for i in range(n))
    return {"bytes": 2 * seen * row + 2 * sum(new) * case["heads"] * case["hd"] * SIZE[case["dtype"]],
            "flops": 4.0 * pairs * case["heads"] * case["hd"]}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _requests(case, seed):
    """Lengths in this seed's order, and a table of pages for each request."""
    total, new = _lengths(case)
    rng = random.Random(seed * 7919 + 13)
    order = list(range(case["batch"]))
    rng.shuffle(order)
    total, new = [total[i] for i in order], [new[i] for i in order]
    P = case["page"]
    n_pages = _n_pages(case)
    pages = list(range(n_pages))
    rng.shuffle(pages)
    width = max(-(-t // P) for t in total)
    tables, at = [], 0
    for t in total:
        k = -(-t // P)
        tables.append(pages[at:at + k] + [-1] * (width - k))
        at += k
    return total, new, tables, pages[at:], n_pages


def _offsets(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(TORCH[dtype])


def _pool(g, shape):
    """e4m3 values and power-of-two scales as ``kv_store_paged`` leaves them for
    normal keys whose size differs from head to head."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    x *= torch.exp2(torch.rand(shape[:2] + (1, 1), generator=g, device=DEV) * 2 - 1)
    scale = _power(x.abs().amax((2, 3)))
    return (x / scale[:, :, None, None]).to(E4M3), scale


def _power(amax):
    """2^e, e the least whole number with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax.double())  # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.exp2(e.clamp(min=-100).double()).where(amax > 0, 2.0 ** -100).float()


def _inputs(case, seed):
    op, g = case["op"], _gen(seed)
    if op == "sample":
        B, V = case["batch"], case["vocab"]
        # a model's logits: a wide bulk and a few likely tokens; every fifth row
        # under a grammar's mask
        x = torch.randn((B, V), generator=g, device=DEV) * 2.0
        hot = torch.randint(0, V, (B, min(V, 24)), generator=g, device=DEV)
        x.scatter_add_(1, hot, torch.rand(hot.shape, generator=g, device=DEV) * 9.0)
        x[::5] = torch.where(torch.rand((len(x[::5]), V), generator=g, device=DEV) < 0.5, -math.inf, x[::5])
        s = {"logits": x.to(TORCH[case["dtype"]]), "u": torch.rand(B, generator=g, device=DEV)}
        if case["mixed"]:
            pick = lambda vals: torch.tensor(vals, device=DEV)[torch.randint(0, len(vals), (B,), generator=g, device=DEV)]  # noqa: E731
            s.update(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.4]), top_k=pick([0, 0, 1, 20, 50, 1000]).int(),
                     top_p=pick([1.0, 1.0, 0.9, 0.95, 0.3]), min_p=pick([0.0, 0.0, 0.0, 0.02, 0.1]))
        else:
            s.update(temperature=torch.full((B,), 0.8, device=DEV), top_k=None,
                     top_p=torch.full((B,), 0.95, device=DEV), min_p=None)
        return s
    total, new, tables, spare, n_pages = _requests(case, seed)
    P = case["page"]
    if op == "plan":
        old = [t - n for t, n in zip(total, new)]
        free = [p for t, o, row in zip(total, old, tables) for p in row[-(-o // P):-(-t // P)]] + spare
        random.Random(seed).shuffle(free)
        held = [[p if i < -(-o // P) else -1 for i, p in enumerate(row)] for o, row in zip(old, tables)]
        return {"lens": _i32(old), "new": _i32(new), "free": _i32(free), "tables": _i32(held), "n_pages": n_pages}
    cu = _offsets(new)
    if op == "store":
        k_cache, k_scale = _pool(g, (n_pages, case["kv"], P, case["hd"]))
        v_cache, v_scale = _pool(g, (n_pages, case["kv"], case["hd"], P))
        # keys and values as views into one projection's rows
        rows = _normal(g, (cu[-1], 2, case["kv"], case["hd"]), case["dtype"])
        slots = [tables[b][p // P] * P + p % P for b in range(len(new)) for p in range(total[b] - new[b], total[b])]
        return {"k": rows[:, 0], "v": rows[:, 1], "slots": _i32(slots), "k_cache": k_cache, "v_cache": v_cache,
                "k_scale": k_scale, "v_scale": v_scale}
    k_cache, k_scale = _pool(g, (n_pages, case["kv"], P, case["hd"]))
    v_cache, v_scale = _pool(g, (n_pages, case["kv"], case["hd"], P))
    return {"q": _normal(g, (cu[-1], case["heads"], case["hd"]), case["dtype"]), "k_cache": k_cache, "v_cache": v_cache,
            "k_scale": k_scale, "v_scale": v_scale, "tables": _i32(tables), "lens": _i32(total), "cu": _i32(cu),
            "max_q": max(new), "max_len": max(total)}


_backend = None


def _hip():
    global _backend
    if _backend is None:
        from munet_amd.backend import HipBackend
        _backend = HipBackend(torch.cuda.current_device())
    return _backend


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=dict(case))
    op = case["op"]
    if op == "plan":
        B, n = case["batch"], int(s["new"].sum())
        s.update(total=torch.empty(B, dtype=torch.int32, device=DEV), cu=torch.empty(B + 1, dtype=torch.int32, device=DEV),
                 slots=torch.empty(n, dtype=torch.int32, device=DEV), positions=torch.empty(n, dtype=torch.int32, device=DEV),
                 used=torch.empty(1, dtype=torch.int32, device=DEV))
    elif op == "attend":
        s["out"] = torch.empty_like(s["q"])
    elif op == "sample":
        s["ids"] = torch.empty(case["batch"], dtype=torch.int32, device=DEV)
        s["logprob"] = torch.empty(case["batch"], dtype=torch.float32, device=DEV)
    # the buffer that a server keeps for its attention's and its sampler's partial results
    s["workspace"] = None
    if own and op == "attend":
        n = _hip().attention_paged_workspace(s["q"], s["k_cache"], s["lens"], s["max_q"], s["max_len"], window=case["window"])
        s["workspace"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    elif own and op == "sample":
        s["workspace"] = torch.empty(_hip().sample_workspace(s["logits"]), dtype=torch.uint8, device=DEV)
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


# ---- the framework's calls -----------------------------------------------------

def _own_plan(s):
    _hip().page_plan(s["lens"], s["new"], s["free"], s["tables"], s["total"], s["cu"], s["slots"], s["positions"], s["used"],
                     s["case"]["page"], s["n_pages"])
    return {k: s[k] for k in ("tables", "total", "cu", "slots", "positions", "used")}


def _own_store(s):
    _hip().kv_store_paged(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _own_attend(s):
    _hip().attention_paged(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"], s["lens"], s["cu"],
                           s["out"], s["max_q"], s["max_len"], causal=True, window=s["case"]["window"], workspace=s["workspace"])
    return s["out"]


def _own_sample(s):
    _hip().sample(s["logits"], s["u"], s["ids"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                  min_p=s["min_p"], logprob=s["logprob"], workspace=s["workspace"])
    return {"ids": s["ids"], "logprob": s["logprob"]}


_OWN = {"plan": _own_plan, "store": _own_store, "attend": _own_attend, "sample": _own_sample}


# ---- the plain forms -------------------------------------------------------------

def _plain_plan(s):
    P = s["case"]["page"]
    lens, new, free = s["lens"].long(), s["new"].long(), s["free"].long()
    total = lens + new
    have, need = (lens + P - 1) // P, (total + P - 1) // P
    end = torch.cumsum(need - have, 0)
    first = end - (need - have)
    p = torch.arange(s["tables"].shape[1], device=DEV)
    fresh = (p >= have[:, None]) & (p < need[:, None])
    at = (first[:, None] + p - have[:, None]).clamp(0, len(free) - 1)
    s["tables"].copy_(torch.where(fresh, free[at].int(), s["tables"]))
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), torch.cumsum(new, 0)])
    t = torch.arange(s["slots"].shape[0], device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = lens[b] + t - cu[b]
    slots = s["tables"].long()[b, pos // P] * P + pos % P
    return {"tables": s["tables"], "total": total.int(), "cu": cu.int(), "slots": slots.int(), "positions": pos.int(),
            "used": end[-1:].int()}


def _plain_store_one(x, slots, cache, scale, token_dim):
    """One of the two caches: the scale of each page that gets tokens, its older
    tokens in that scale, the new ones beside them."""
    P = cache.shape[token_dim]
    page, place = slots // P, slots % P
    amax = x.float().abs().amax(2)                                      # [n, heads]
    most = torch.zeros_like(scale).index_reduce_(0, page, amax, "amax")
    first = torch.full((cache.shape[0],), P, device=DEV).index_reduce_(0, page, place, "amin")
    touched = (first < P)[:, None]
    want = _power(most)
    now = torch.where(touched, torch.where((first == 0)[:, None], want, torch.maximum(scale, want)), scale)
    grown = torch.unique(page)
    ratio = (scale / now)[grown][:, :, None, None]
    older = (torch.arange(P, device=DEV) < first[grown][:, None])       # [pages, P]
    older = older[:, None, :, None] if token_dim == 2 else older[:, None, None, :]
    held = cache[grown].float()
    cache.view(torch.uint8)[grown] = torch.where(older, (held * ratio), held).to(E4M3).view(torch.uint8)
    q = (x.float() / now[page][:, :, None]).to(E4M3).view(torch.uint8)  # [n, heads, hd]
    if token_dim == 2:
        cache.view(torch.uint8)[page, :, place] = q
    else:
        cache.view(torch.uint8)[page, :, :, place] = q
    scale.copy_(now)


def _plain_store(s):
    slots = s["slots"].long()
    _plain_store_one(s["k"], slots, s["k_cache"], s["k_scale"], 2)
    _plain_store_one(s["v"], slots, s["v_cache"], s["v_scale"], 3)
    return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _plain_attend(s):
    c = s["case"]
    B, H, KV, hd, P = c["batch"], c["heads"], c["kv"], c["hd"], c["page"]
    lens, cu, tables = s["lens"].long(), s["cu"].long(), s["tables"].long().clamp(min=0)
    n_q, T = s["max_q"], tables.shape[1] * P
    # every request's pages as rows of keys and values: [B, KV, T, hd]
    k = s["k_cache"][tables].float() * s["k_scale"][tables][..., None, None]
    v = s["v_cache"][tables].float() * s["v_scale"][tables][..., None, None]
    k = k.transpose(1, 2).reshape(B, KV, T, hd)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, KV, T, hd)
    # queries padded to the longest request's: [B, KV, n_q * group, hd]
    i = torch.arange(n_q, device=DEV)
    count = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].reshape(B, n_q, KV, H // KV, hd).permute(0, 2, 1, 3, 4)
    pos = (lens - count)[:, None] + i                                   # [B, n_q]
    j = torch.arange(T, device=DEV)
    seen = (j <= pos[..., None]) & (j < lens[:, None, None])
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    scores = torch.matmul(q.reshape(B, KV, -1, hd), k.transpose(2, 3).contiguous()).reshape(B, KV, n_q, -1, T)
    scores = (scores * (1.0 / math.sqrt(hd))).masked_fill(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    w = torch.exp(scores - top)
    v = v.masked_fill(~(j < lens[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(w.reshape(B, KV, -1, T), v).reshape(B, KV, n_q, -1, hd)
    o = o / w.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n_q, H, hd)
    live = i < count[:, None]
    s["out"].copy_(o[live].to(s["q"].dtype))
    return s["out"]


def _plain_sample(s):
    x = s["logits"].double()
    B, V = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    row = lambda v, off: torch.full((B, 1), off, dtype=torch.float64, device=DEV) if v is None else v.double()[:, None]  # noqa: E731
    T, k, p, m = row(s["temperature"], 1.0), row(s["top_k"], 0.0), row(s["top_p"], 1.0), row(s["min_p"], 0.0)
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = xs[:, :1]
    w = torch.where(xs == top, 1.0, torch.exp((xs - top) / torch.where(T > 0, T, 1.0)))
    rank = torch.arange(V, device=DEV)[None]
    n_k = torch.where((k > 0) & (k < V), k, float(V))
    cum = torch.cumsum(torch.where(rank < n_k, w, 0.0), 1)
    n_p = torch.where(p < 1, (cum < p * cum[:, -1:]).sum(1, keepdim=True) + 1.0, float(V))
    n_m = torch.where(m > 0, (w >= m.clamp(max=1.0)).sum(1, keepdim=True).double(), float(V))
    n = torch.minimum(torch.minimum(n_k, n_p), n_m).clamp(min=1)
    n = torch.where(T > 0, n, 1.0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(rank < n, w, 0.0))  # back in index order
    cum = torch.cumsum(kept, 1)
    total = cum[:, -1:]
    ids = (cum <= s["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=V - 1)
    # a row with nothing to draw from has no token
    none = top == -math.inf
    logprob = torch.log(kept.gather(1, ids) / total)
    return {"ids": torch.where(none, -1, ids)[:, 0].int(), "logprob": torch.where(none, -math.inf, logprob)[:, 0].float()}


_PLAIN = {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend, "sample": _plain_sample}


# ---- the definitions in 64 bits ------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "plan":
        return None  # whole numbers: the plain form's are right or wrong
    if op == "store":
        return _exact_store(case, s)
    if op == "attend":
        return _exact_attend(case, s)
    return _exact_sample(case, s)


def _exact_scale(amax):
    """The least power of two whose 448-fold holds amax, by counting up and down."""
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / E4M3_MAX))
    e = torch.where(amax > E4M3_MAX * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)
    return torch.where(amax > 0, torch.exp2(e.clamp(min=-100)), 2.0 ** -100)


def _exact_e4m3(x):
    """Nearest e4m3 value, ties to the even one, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_store(case, s):
    P, found = case["page"], {}
    slots = s["slots"].cpu().long()
    runs, page = [], (slots // P).tolist()
    at = 0
    while at < len(page):  # tokens of one page follow each other
        end = at
        while end < len(page) and page[end] == page[at]:
            end += 1
        runs.append((page[at], int(slots[at]) % P, at, end))
        at = end
    if len(runs) > 4000:
        return None
    for name, x, dim in (("k", s["k"], 2), ("v", s["v"], 3)):
        cache, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        for g, first, a, b in runs:
            new = x[a:b].double()
            want = _exact_scale(new.abs().amax((0, 2)))
            now = want if first == 0 else torch.maximum(scale[g], want)
            held = cache[g] if dim == 2 else cache[g].transpose(1, 2)      # [heads, P, hd]
            held[:, :first] = _exact_e4m3(held[:, :first] * (scale[g] / now)[:, None, None])
            held[:, first:first + b - a] = _exact_e4m3(new.transpose(0, 1) / now[:, None, None])
            scale[g] = now
        found[name + "_cache"], found[name + "_scale"] = cache, scale
    return found


def _exact_attend(case, s):
    group, hd, P = case["heads"] // case["kv"], case["hd"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    for b, length in enumerate(lens):
        first, n = cu[b], cu[b + 1] - cu[b]
        pages = s["tables"][b, :-(-length // P)].long()
        pos = torch.arange(length - n, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)[None]
        hidden = (j > pos) | ((j <= pos - case["window"]) if case["window"] else (j < 0))
        for h in range(case["kv"]):
            k = (s["k_cache"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, hd)[:length]
            v = (s["v_cache"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, hd)[:length]
            q = s["q"][first:first + n, h * group:(h + 1) * group].double()
            a = torch.tensordot(q, k, dims=([2], [1])) / math.sqrt(hd)    # [n, group, length]
            a = torch.softmax(a.masked_fill(hidden[:, None], -math.inf), -1)
            out[first:first + n, h * group:(h + 1) * group] = torch.tensordot(a, v, dims=([2], [0]))
    return out


def _exact_sample(case, s):
    """One row at a time, the tokens in the order of the definition."""
    x = s["logits"].double().cpu()
    ids, logprob = [], []
    at = lambda name, r, off: off if s[name] is None else float(s[name][r])  # noqa: E731
    for r in range(x.shape[0]):
        T, k, p, m = at("temperature", r, 1.0), int(at("top_k", r, 0)), at("top_p", r, 1.0), at("min_p", r, 0.0)
        best = float(x[r].max())
        if best == -math.inf:
            ids.append(-1)
            logprob.append(-math.inf)
            continue
        if T <= 0:
            ids.append(int(torch.nonzero(x[r] == best)[0]))
            logprob.append(0.0)
            continue
        w = torch.exp((x[r] - best) / T)
        order = torch.argsort(-x[r], stable=True)
        if 0 < k < len(order):
            order = order[:k]
        n = len(order)
        if p < 1:
            cum = torch.cumsum(w[order], 0)
            n = min(n, int((cum < p * cum[-1]).sum()) + 1)
        if m > 0:
            n = min(n, int((w >= min(m, 1.0)).sum()))
        keep, _ = torch.sort(order[:max(1, n)])
        cum = torch.cumsum(w[keep], 0)
        i = min(int((cum <= float(s["u"][r]) * float(cum[-1])).sum()), len(keep) - 1)
        ids.append(int(keep[i]))
        logprob.append(math.log(float(w[keep[i]]) / float(cum[-1])))
    return {"ids": None, "logprob": torch.tensor(logprob, dtype=torch.float64)}
