"""Operators of a decoder layer that serves in 8 bits: rotary positions, keys
that are rotated on their way into the paged cache, and matrix products in 8-bit
integers.

A program that serves a decoder with rotary positions works out the angles of a
step's tokens once (``rotary_table``) and uses them in every layer: to rotate
queries and keys (``rotary``), or to rotate the queries and store the rotated
keys and the values in the paged 8-bit cache in one call
(``kv_store_rotary_paged``).  Its Linear layers round each token's values to 8
bits (``quantize_rows``, ``dequantize_rows`` the way back) and multiply them
with weights that were rounded so once, a scale for each token and each output
channel (``linear_i8``).

Layouts.  A table is [tokens, pairs, 2]: the cosine and sine of each pair's
angle.  A page holds P tokens of every key/value head: ``k_cache`` [pages, Hkv, P,
hd] and ``v_cache`` [pages, Hkv, hd, P] in e4m3, ``k_scale`` and ``v_scale``
[pages, Hkv] in float32, powers of two.  A slot is page * P + place.
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
        # the angles of one decode step, a token per request
        {"name": "angles_step", "op": "angles", "tokens": 64, "rot": 128, "far": 8192, "factor": 1.0},
        # the angles of a queue of long documents, frequencies stretched eight times
        {"name": "angles_documents", "op": "angles", "tokens": 17000, "rot": 128, "far": 1000000, "factor": 8.0},
        # a decode step on heads of the repository's decoder (12 of 64), queries and
        # keys as they lie in one projection's rows: latency
        {"name": "rotate_step", "op": "rotate", "dtype": "float16", "tokens": 4, "heads": 24, "behind": 12, "hd": 64, "rot": 64,
         "interleaved": False},
        # prompts of a serving batch, neighbours paired
        {"name": "rotate_prompts", "op": "rotate", "dtype": "bfloat16", "tokens": 16500, "heads": 40, "behind": 8, "hd": 128,
         "rot": 128, "interleaved": True},
        # one token of each request into its page
        {"name": "append_step", "op": "append", "dtype": "bfloat16", "batch": 64, "new": 1, "len": 4096, "page": 64, "heads": 32,
         "kv": 8, "hd": 128, "rot": 128, "interleaved": False, "spread": 1},
        # prompts of uneven lengths, some behind a cached prefix
        {"name": "append_prompts", "op": "append", "dtype": "bfloat16", "batch": 12, "new": 2500, "len": 300, "page": 64,
         "heads": 32, "kv": 8, "hd": 128, "rot": 128, "interleaved": False, "spread": 2},
        # short ragged prompts in single precision, a part of each head rotated
        {"name": "append_partial", "op": "append", "dtype": "float32", "batch": 16, "new": 237, "len": 40, "page": 16, "heads": 12,
         "kv": 12, "hd": 64, "rot": 24, "interleaved": True, "spread": 3},
        # a decode step's activations to 8 bits and back
        {"name": "rows_step", "op": "rows", "dtype": "bfloat16", "rows": 64, "cols": 4096},
        # a prompt batch's
        {"name": "rows_prompts", "op": "rows", "dtype": "bfloat16", "rows": 8192, "cols": 8192},
        # one user's next token, the repository's decoder's q/k/v product: latency
        {"name": "linear_one", "op": "linear", "dtype": "bfloat16", "rows": 1, "k": 768, "n": 2304, "bias": True, "act": 0,
         "resid": False},
        # a decode step of a serving batch: the weights' bytes
        {"name": "linear_batch", "op": "linear", "dtype": "bfloat16", "rows": 64, "k": 4096, "n": 12800, "bias": False, "act": 0,
         "resid": False},
        # prompts: the matrix work, with the residual that follows a layer's last product
        {"name": "linear_prompts", "op": "linear", "dtype": "bfloat16", "rows": 8192, "k": 8192, "n": 8192, "bias": True, "act": 0,
         "resid": True},
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
    op = rng.choice(["angles", "rotate", "rotate", "append", "append", "append", "rows", "rows", "linear", "linear", "linear"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "angles":
        return {"op": op, "tokens": _log(rng, 1, 40000), "rot": 2 * _log(rng, 1, 128), "far": _log(rng, 100, 10000000),
                "factor": rng.choice([1.0, 1.0, 4.0, 32.0])}
    if op == "rows":
        return {"op": op, "dtype": dtype, "rows": _log(rng, 1, 20000), "cols": _log(rng, 1, 30000)}
    if op == "linear":
        return {"op": op, "dtype": dtype, "rows": rng.choice([_log(rng, 1, 64), _log(rng, 1, 10000)]), "k": _log(rng, 16, 16384),
                "n": _log(rng, 16, 32000), "bias": rng.random() < 0.5, "act": rng.choice([0, 0, 1, 2]), "resid": rng.random() < 0.3}
    hd = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    c = {"op": op, "dtype": dtype, "hd": hd, "rot": rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]),
         "interleaved": rng.random() < 0.4}
    if op == "rotate":
        c.update(tokens=_log(rng, 1, 20000), heads=rng.choice([1, 4, 5, 24, 40]), behind=rng.choice([0, 0, 1, 8]))
        return c
    group, kv = rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 8, 12])
    c.update(batch=_log(rng, 1, 256), page=rng.choice([16, 32, 64, 64, 128, 256]), spread=rng.randrange(1000), heads=group * kv,
             kv=kv, new=rng.choice([1, 1, _log(rng, 1, 4000)]), len=_log(rng, 1, 4000))
    return c


def _cost(case):
    """Work of a case in the plain form's terms, to keep draws below the listed ones."""
    w = work(case)
    held = _n_pages(case) * case["page"] * case["kv"] * case["hd"] * 8.0 if case["op"] == "append" else 0.0
    return w["bytes"] + w["flops"] / 200.0 + held


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
        old = case["len"] if i == 0 else int(case["len"] * rng.random())
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
    if op == "angles":
        pairs = case["tokens"] * case["rot"] // 2
        return {"bytes": 4 * case["tokens"] + 4 * case["rot"] + 8 * pairs, "flops": 4.0 * pairs}
    if op == "rows":
        n = case["rows"] * case["cols"]
        # there and back: the values, their 8 bits written and read, the values again
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 2 * n + 8 * case["rows"], "flops": 4.0 * n}
    if op == "linear":
        M, N, K, e = case["rows"], case["n"], case["k"], SIZE[case["dtype"]]
        return {"bytes": M * K + N * K + 4 * (M + N) + M * N * e * (2 if case["resid"] else 1) + (N * e if case["bias"] else 0),
                "flops": 2.0 * M * N * K}
    e = SIZE[case["dtype"]]
    if op == "rotate":
        n = case["tokens"]
        return {"bytes": 2 * n * case["heads"] * case["hd"] * e + 4 * n * case["rot"], "flops": 3.0 * n * case["heads"] * case["rot"]}
    n = sum(_lengths(case)[1])
    row, qrow = case["kv"] * case["hd"], case["heads"] * case["hd"]
    return {"bytes": n * (2 * row * (e + 1) + 2 * qrow * e + 4 * case["rot"] + 4),
            "flops": n * (4.0 * row + 3.0 * case["rot"] * (case["heads"] + case["kv"]))}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(TORCH[dtype])


def _frequencies(rot, factor):
    """Frequencies of a model of base 10000, those that turn less than 32 times in
    its 4096 trained positions stretched by ``factor`` (all of it below one turn)."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if factor != 1.0:
        keep = ((4096 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.to(DEV), 1.0 if factor == 1.0 else 1.0 + 0.1 * math.log(factor)


def _angles(positions, rot):
    """The table of a step's tokens, as its program keeps it for all layers."""
    a = positions.double()[:, None] * _frequencies(rot, 1.0)[0]
    return torch.stack([torch.cos(a), torch.sin(a)], -1).float()


def _activations(g, rows, cols):
    """A layer's activations: a bulk near zero, some channels far larger, and tokens
    that differ in size."""
    x = torch.randn((rows, cols), generator=g, device=DEV, dtype=torch.float32)
    x *= torch.exp2(torch.rand((rows, 1), generator=g, device=DEV) * 4 - 2)
    return x * torch.where(torch.rand((1, cols), generator=g, device=DEV) < 0.02, 12.0, 1.0)


def _to_8_bits(x):
    a = x.abs().amax(1, keepdim=True).clamp(min=127 * 2.0 ** -126).double()
    return torch.round(127 * x.double() / a).to(torch.int8), (a / 127).float()[:, 0]


def _pool(g, shape):
    """e4m3 values and power-of-two scales as the cache's writes leave them for
    normal keys whose size differs from head to head."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    x *= torch.exp2(torch.rand(shape[:2] + (1, 1), generator=g, device=DEV) * 2 - 1)
    scale = _power(x.abs().amax((2, 3)))
    return (x / scale[:, :, None, None]).to(E4M3), scale


def _power(amax):
    """2^e, e the least whole number with amax <= 448 * 2^e, from -100 on."""
    m, e = torch.frexp(amax.double())  # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.exp2(e.clamp(min=-100).double()).where(amax > 0, 2.0 ** -100).float()


def _inputs(case, seed):
    op, g = case["op"], _gen(seed)
    if op == "angles":
        # runs of neighbouring positions, as prompts and their chunks have them
        n, run = case["tokens"], max(1, case["tokens"] // 7)
        first = torch.randint(0, case["far"], (-(-n // run), 1), generator=g, device=DEV)
        freq, magnitude = _frequencies(case["rot"], case["factor"])
        return {"positions": (first + torch.arange(run, device=DEV)).reshape(-1)[:n].int(), "freq": freq, "magnitude": magnitude}
    if op == "rotate":
        rows = _normal(g, (case["tokens"], case["heads"] + case["behind"], case["hd"]), case["dtype"])
        positions = torch.randint(0, 8192, (case["tokens"],), generator=g, device=DEV)
        return {"x": rows[:, :case["heads"]], "table": _angles(positions, case["rot"])}
    if op == "rows":
        return {"x": _activations(g, case["rows"], case["cols"]).to(TORCH[case["dtype"]])}
    if op == "linear":
        M, N, K = case["rows"], case["n"], case["k"]
        x, sx = _to_8_bits(_activations(g, M, K))
        w, sw = _to_8_bits(torch.randn((N, K), generator=g, device=DEV) * (0.7 / math.sqrt(K)))
        return {"x": x, "sx": sx, "w": w, "sw": sw, "bias": _normal(g, (N,), case["dtype"]) if case["bias"] else None,
                "resid": _normal(g, (M, N), case["dtype"]) if case["resid"] else None}
    total, new = _lengths(case)
    P, n_pages = case["page"], _n_pages(case)
    rng = random.Random(seed * 7919 + 13)
    pages = list(range(n_pages))
    rng.shuffle(pages)
    slots, positions, at = [], [], 0
    for t, n in zip(total, new):
        slots += [pages[at + p // P] * P + p % P for p in range(t - n, t)]
        positions += range(t - n, t)
        at += -(-t // P)
    k_cache, k_scale = _pool(g, (n_pages, case["kv"], P, case["hd"]))
    v_cache, v_scale = _pool(g, (n_pages, case["kv"], case["hd"], P))
    # queries, keys and values as views into one projection's rows
    H, KV = case["heads"], case["kv"]
    rows = _normal(g, (len(slots), H + 2 * KV, case["hd"]), case["dtype"])
    return {"q": rows[:, :H], "k": rows[:, H:H + KV], "v": rows[:, H + KV:], "table": _angles(_i32(positions), case["rot"]),
            "slots": _i32(slots), "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale}


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
    empty = lambda shape, t: torch.empty(shape, dtype=t, device=DEV)  # noqa: E731
    # the buffers that a program keeps for what the calls write
    if op == "angles":
        s["table"] = empty((case["tokens"], case["rot"] // 2, 2), torch.float32)
    elif op == "rotate":
        s["out"] = empty(s["x"].shape, s["x"].dtype)
    elif op == "append":
        s["q_out"] = empty(s["q"].shape, s["q"].dtype)
    elif op == "rows":
        s.update(q=empty(s["x"].shape, torch.int8), scale=empty((case["rows"],), torch.float32), values=torch.empty_like(s["x"]))
    else:
        s["out"] = empty((case["rows"], case["n"]), TORCH[case["dtype"]])
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


# ---- the framework's calls -----------------------------------------------------

def _own_angles(s):
    _hip().rotary_table(s["positions"], s["freq"], s["table"], magnitude=s["magnitude"])
    return s["table"]


def _own_rotate(s):
    _hip().rotary(s["x"], s["table"], s["out"], interleaved=s["case"]["interleaved"])
    return s["out"]


def _own_append(s):
    _hip().kv_store_rotary_paged(s["k"], s["v"], s["table"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                 q=s["q"], q_out=s["q_out"], interleaved=s["case"]["interleaved"])
    return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale", "q_out")}


def _own_rows(s):
    _hip().quantize_rows(s["x"], s["q"], s["scale"])
    _hip().dequantize_rows(s["q"], s["scale"], s["values"])
    return {"values": s["values"], "scale": s["scale"]}


def _own_linear(s):
    _hip().linear_i8(s["x"], s["sx"], s["w"], s["sw"], s["out"], bias=s["bias"], act=s["case"]["act"], resid=s["resid"])
    return s["out"]


_OWN = {"angles": _own_angles, "rotate": _own_rotate, "append": _own_append, "rows": _own_rows, "linear": _own_linear}


# ---- the plain forms -------------------------------------------------------------

def _plain_angles(s):
    # far positions: angles of a million turns, in 64 bits
    a = s["positions"].double()[:, None] * s["freq"]
    s["table"].copy_(torch.stack([torch.cos(a), torch.sin(a)], -1) * s["magnitude"])
    return s["table"]


def _rotated(x, table, interleaved, out):
    """x with its first pairs turned by the table's angles, in ``out``'s type."""
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    h = table.shape[1]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    y = (a * c - b * s, a * s + b * c)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, x[..., 2 * h:]], -1).to(out)


def _plain_rotate(s):
    s["out"].copy_(_rotated(s["x"].float(), s["table"], s["case"]["interleaved"], s["x"].dtype))
    return s["out"]


def _plain_store_one(x, slots, cache, scale, token_dim):
    """One of the two caches: the scale of each page that gets tokens, its older
    tokens in that scale, the new ones beside them."""
    P = cache.shape[token_dim]
    page, place = slots // P, slots % P
    most = torch.zeros(scale.shape, dtype=x.dtype, device=DEV).index_reduce_(0, page, x.abs().amax(2), "amax")
    first = torch.full((cache.shape[0],), P, device=DEV).index_reduce_(0, page, place, "amin")
    want = _power(most)
    now = torch.where((first == 0)[:, None], want, torch.maximum(scale, want))
    now = torch.where((first < P)[:, None], now, scale)
    got = torch.unique(page)
    older = torch.arange(P, device=DEV) < first[got][:, None]           # [pages, P]
    older = older[:, None, :, None] if token_dim == 2 else older[:, None, None, :]
    held = cache[got].float()
    cache.view(torch.uint8)[got] = torch.where(older, held * (scale / now)[got][:, :, None, None], held).to(E4M3).view(torch.uint8)
    q = (x / now[page][:, :, None]).float().to(E4M3).view(torch.uint8)   # [n, heads, hd]
    if token_dim == 2:
        cache.view(torch.uint8)[page, :, place] = q
    else:
        cache.view(torch.uint8)[page, :, :, place] = q
    scale.copy_(now)


def _plain_append(s):
    slots, inter = s["slots"].long(), s["case"]["interleaved"]
    # in 64 bits: a page's scale goes by its largest key, next to a power of two
    _plain_store_one(_rotated(s["k"].double(), s["table"].double(), inter, torch.float64), slots, s["k_cache"], s["k_scale"], 2)
    _plain_store_one(s["v"].float(), slots, s["v_cache"], s["v_scale"], 3)
    s["q_out"].copy_(_rotated(s["q"].float(), s["table"], inter, s["q"].dtype))
    return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale", "q_out")}


def _plain_rows(s):
    # in 64 bits: which whole number is nearest is decided next to a half
    q, scale = _to_8_bits(s["x"])
    s["scale"].copy_(scale)
    s["values"].copy_(q.float() * scale[:, None])
    return {"values": s["values"], "scale": s["scale"]}


def _plain_linear(s):
    y = torch.matmul(s["x"].float(), s["w"].float().t()) * s["sx"][:, None] * s["sw"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    act = s["case"]["act"]
    if act == 1:
        y = y.clamp(min=0)
    elif act == 2:
        y = y / (1 + torch.exp(-1.702 * y))
    if s["resid"] is not None:
        y = y + s["resid"].float()
    s["out"].copy_(y)
    return s["out"]


_PLAIN = {"angles": _plain_angles, "rotate": _plain_rotate, "append": _plain_append, "rows": _plain_rows, "linear": _plain_linear}


# ---- the definitions in 64 bits ------------------------------------------------

def exact(case, seed):
    return _EXACT[case["op"]](case, _inputs(case, seed))


def _exact_angles(case, s):
    turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device=DEV), torch.outer(s["positions"].double(), s["freq"]))
    return torch.view_as_real(turn)


def _exact_turn(x, table, interleaved):
    """Pairs as complex numbers, times the table's."""
    y, h = x.double().clone(), table.shape[1]
    first = slice(0, 2 * h, 2) if interleaved else slice(0, h)
    second = slice(1, 2 * h, 2) if interleaved else slice(h, 2 * h)
    z = torch.complex(y[..., first], y[..., second]) * torch.view_as_complex(table.double())[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotate(case, s):
    return _exact_turn(s["x"], s["table"], case["interleaved"])


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


def _exact_append(case, s):
    P = case["page"]
    slots = s["slots"].tolist()
    runs, at = [], 0
    while at < len(slots):  # tokens of one page follow each other
        end = at
        while end < len(slots) and slots[end] // P == slots[at] // P:
            end += 1
        runs.append((slots[at] // P, slots[at] % P, at, end))
        at = end
    if len(runs) > 4000:
        return None
    found = {"q_out": _exact_turn(s["q"], s["table"], case["interleaved"])}
    keys = _exact_turn(s["k"], s["table"], case["interleaved"])
    for name, x, dim in (("k", keys, 2), ("v", s["v"], 3)):
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


def _exact_rows(case, s):
    x = s["x"].double()
    step = torch.clamp(torch.amax(torch.abs(x), dim=1), min=127 * 2.0 ** -126) / 127
    whole = torch.round(127 * x / torch.clamp(torch.amax(torch.abs(x), dim=1, keepdim=True), min=127 * 2.0 ** -126))
    return {"values": whole * step[:, None], "scale": step}


def _exact_linear(case, s):
    x, w = s["x"].double() * s["sx"].double()[:, None], s["w"].double() * s["sw"].double()[:, None]
    y = torch.tensordot(x, w, dims=([1], [1]))
    if case["bias"]:
        y += s["bias"].double()
    if case["act"] == 1:
        y = torch.where(y > 0, y, 0.0)
    elif case["act"] == 2:
        y *= torch.sigmoid(1.702 * y)
    if case["resid"]:
        y += s["resid"].double()
    return y


_EXACT = {"angles": _exact_angles, "rotate": _exact_rotate, "append": _exact_append, "rows": _exact_rows, "linear": _exact_linear}
