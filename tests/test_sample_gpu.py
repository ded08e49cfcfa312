"""Sampling on the GPU against the definition in 64 bits, one row at a time.

Tokens are whole numbers and must be equal.  The kernel's sums carry 44 bits
after the largest weight's point and the reference's 52: a draw could differ
only where u falls within about 2^-40 of a border, which none of these (u of 24
bits or less, and borders computed from independent random logits) meets; where
a test puts u or top_p on a border on purpose, all weights are equal, and both
sums are exact.  logprob: float32 of a 64-bit logarithm, half a step (2^-24) of
it and 2^-40 for the sums.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16", "float32"]


@pytest.fixture(scope="module")
def torch(hip):
    import torch as t
    return t


def reference(torch, logits, u, T=None, k=None, p=None, m=None):
    ids, logprob = [], []
    x_all = logits.double().cpu()
    x_all = torch.where(torch.isnan(x_all), -math.inf, x_all)
    at = lambda v, r, off: off if v is None else float(v[r])  # noqa: E731
    for r in range(x_all.shape[0]):
        x, t, kk, pp, mm = x_all[r], at(T, r, 1.0), int(at(k, r, 0)), at(p, r, 1.0), at(m, r, 0.0)
        best = float(x.max())
        if best == -math.inf:
            ids.append(-1)
            logprob.append(-math.inf)
            continue
        if not t > 0:
            ids.append(int((x == best).nonzero()[0]))
            logprob.append(0.0)
            continue
        w = torch.where(x == best, 1.0, torch.exp((x - best) / t))
        w = torch.where(x == -math.inf, 0.0, w)  # (also where T is infinite)
        order = torch.argsort(-x, stable=True)
        order = order[:kk] if 0 < kk < len(order) else order
        n = len(order)
        if pp < 1:
            cum = torch.cumsum(w[order], 0)
            n = min(n, int((cum < max(pp, 0.0) * cum[-1]).sum()) + 1)
        if mm > 0:
            n = min(n, int((w >= min(mm, 1.0)).sum()))
        keep = order[:max(n, 1)].sort().values
        cum = torch.cumsum(w[keep], 0)
        uu = at(u, r, 0.0)
        i = int((cum <= (uu if uu > 0 else 0.0) * float(cum[-1])).sum())
        if i >= len(keep):  # u = 1: the last that weighs anything
            i = int(w[keep].nonzero()[-1])
        ids.append(int(keep[i]))
        logprob.append(math.log(float(w[keep[i]])) - math.log(float(cum[-1])))
    return ids, torch.tensor(logprob, dtype=torch.float64)


def run(torch, hip, logits, u, T=None, k=None, p=None, m=None, what=""):
    B = logits.shape[0]
    f = lambda v: None if v is None else torch.as_tensor(v, dtype=torch.float32).cuda()  # noqa: E731
    u, T, p, m = f(u), f(T), f(p), f(m)
    k = None if k is None else torch.as_tensor(k, dtype=torch.int32).cuda()
    out = torch.full((B,), -5, dtype=torch.int32, device="cuda")
    lp = torch.full((B,), 3.0, device="cuda")
    print(f"sample {what} {logits.dtype} {tuple(logits.shape)}", flush=True)
    hip.sample(logits, u, out, temperature=T, top_k=k, top_p=p, min_p=m, logprob=lp)
    ids, logprob = reference(torch, logits, u, T, k, p, m)
    assert out.tolist() == ids, what
    lp = lp.double().cpu()
    fin = torch.isfinite(logprob)
    assert torch.equal(torch.isfinite(lp), fin)
    assert bool(((lp - logprob)[fin].abs() <= logprob[fin].abs() * 2.0 ** -24 + 2.0 ** -40).all()), what
    return out


def logits_like(torch, B, V, dtype, seed=0, scale=3.0):
    return (torch.randn((B, V), generator=torch.Generator().manual_seed(seed)) * scale).to(getattr(torch, dtype)).cuda()


def uniform(torch, B, seed=1):
    return torch.rand(B, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 511, 513, 4096, 4097, 32000, 50257])
def test_plain_draws(torch, hip, dtype, V):
    B = 7
    run(torch, hip, logits_like(torch, B, V, dtype, V), uniform(torch, B, V), what="no filter")
    run(torch, hip, logits_like(torch, B, V, dtype, V + 1), uniform(torch, B, V), T=[0.0, 0.3, 1.0, 5.0, 1e-30, 1e30, -1.0], what="temperature")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 700, 5000, 32000])
def test_filters(torch, hip, dtype, V):
    """Every combination, ties included (16-bit logits repeat values)."""
    ks, ps, ms = [0, 1, 2, 50, 1000], [1.0, 0.95, 0.5, 0.01, 0.0], [0.0, 0.05, 0.5, 1.0]
    combos = [(k, p, m) for k in ks for p in ps for m in ms]
    B = len(combos)
    x = logits_like(torch, B, V, dtype, V, 2.0)
    run(torch, hip, x, uniform(torch, B), T=[0.5 + (i % 4) * 0.5 for i in range(B)], k=[c[0] for c in combos],
        p=[c[1] for c in combos], m=[c[2] for c in combos], what="filters")
    run(torch, hip, x, uniform(torch, B, 5), k=[c[0] for c in combos], what="top-k alone")
    run(torch, hip, x, uniform(torch, B, 6), p=[c[1] for c in combos], what="top-p alone")
    run(torch, hip, x, uniform(torch, B, 7), m=[c[2] for c in combos], what="min-p alone")


@pytest.mark.parametrize("V", [200, 9000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(torch, hip, dtype, V):
    """Few distinct values, zeros of both signs: the lower index is kept."""
    g = torch.Generator().manual_seed(V)
    x = torch.randint(0, 3, (40, V), generator=g).float()
    x = torch.where((x == 0) & (torch.rand((40, V), generator=g) < 0.5), -0.0, x).to(getattr(torch, dtype)).cuda()
    run(torch, hip, x, uniform(torch, 40), T=[1.0] * 40, k=[1 + (7 * i) % V for i in range(40)], p=[1.0 if i % 2 else 0.7 for i in range(40)], what="ties")
    run(torch, hip, torch.zeros_like(x), [i / 40 for i in range(40)], what="all equal")
    run(torch, hip, torch.zeros_like(x), [i / 64 for i in range(40)], p=[0.5] * 40, what="all equal, half kept")
    run(torch, hip, torch.full_like(x, -0.0), [0.0] * 40, T=[0.0] * 40, what="all equal, greedy")


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(torch, hip, dtype):
    """-inf, the type's lowest value, +inf and NaN; rows that leave one token, and none."""
    V, B = 3000, 12
    x = logits_like(torch, B, V, dtype)
    low = torch.finfo(x.dtype).min
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :2999] = -math.inf
    x[3, 1:] = math.nan
    x[4] = low
    x[5, ::2] = low
    x[6, ::3] = -math.inf
    x[7, 17] = math.inf
    x[8, 17] = x[8, 900] = math.inf
    x[9, 5:2900] = math.nan
    x[10] = -math.inf
    x[10, 1234] = low
    for kw in (dict(), dict(k=[40] * B), dict(p=[0.9] * B), dict(k=[2500] * B, p=[0.99] * B, m=[1e-6] * B), dict(T=[0.0] * B)):
        out = run(torch, hip, x, uniform(torch, B), what=f"masks {sorted(kw)}", **kw)
        assert out[0] == -1 and out[1] == -1 and out[2] == 2999 and out[3] == 0 and out[10] == 1234


@pytest.mark.parametrize("dtype", DTYPES)
def test_ends_of_the_range(torch, hip, dtype):
    """u of 0, just below 1, 1 and outside; settings outside their ranges."""
    x = logits_like(torch, 6, 1000, dtype)
    x[:, 0] = x[:, -1] = -math.inf
    run(torch, hip, x, [0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, 0.5], what="u")
    run(torch, hip, x, uniform(torch, 6), T=[math.nan, math.inf, 1.0, 1.0, 1.0, 1.0], k=[-3, 0, 2 ** 31 - 1, 1000, 999, 5],
        p=[-1.0, 2.0, -1.0, 0.999, 1.0, -0.5], m=[-1.0, 5.0, 0.0, -0.0, 2.0, 0.1], what="settings")


@pytest.mark.parametrize("V", [300, 6000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_tokens_at_any_temperature(torch, hip, dtype, V):
    """-inf is never drawn, however flat the rest; without a limit all others are alike (sums exact)."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn((8, V), generator=g).to(getattr(torch, dtype))
    x[:, torch.rand(V, generator=g) < 0.6] = -math.inf
    x[0, 1:] = -math.inf
    u = [0.0, 0.25, 0.5, 0.75, 0.9375, 0.0078125, 0.998046875, 1.0]
    for T in (1e37, 3e38, math.inf):
        for k, p in ((None, None), ([V] * 8, None), ([V // 4] * 8, None), (None, [0.625] * 8)):
            run(torch, hip, x.cuda(), u, [T] * 8, k, p, what=f"T {T} k {k and k[0]} p {p and p[0]}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_apart_and_unaligned(torch, hip, dtype):
    """Rows as a slice of wider ones, at every alignment."""
    wide = logits_like(torch, 5, 1013, dtype)
    for off in range(0, 9):
        x = wide[:, off:off + 1000 - off]
        run(torch, hip, x, uniform(torch, 5), T=[0.7] * 5, k=[30] * 5, p=[0.9] * 5, what=f"offset {off}")


def test_long_rows(torch, hip):
    """More tokens than weights of 44 bits allow, and groups of more than one step."""
    for V in (600001, 1 << 20):
        run(torch, hip, logits_like(torch, 2, V, "float32"), uniform(torch, 2), T=[1.0, 0.7], k=[0, 5000], p=[0.9, 0.9], what="long")
    run(torch, hip, logits_like(torch, 3, 200000, "bfloat16", scale=0.001), [0.1, 0.5, 0.9], p=[0.5, 1.0, 0.99], what="flat")


def test_many_rows(torch, hip):
    run(torch, hip, logits_like(torch, 600, 130, "float16"), uniform(torch, 600), k=[5] * 600, what="many")


def test_frequencies(torch, hip):
    """u on a grid of n numbers draws each token round(n p) times, to within the grid's two ends."""
    n = 4096
    x = torch.randn((1, 50), generator=torch.Generator().manual_seed(3)).repeat(n, 1).cuda()
    out = torch.empty(n, dtype=torch.int32, device="cuda")
    hip.sample(x, ((torch.arange(n) + 0.5) / n).cuda(), out)
    want = torch.softmax(x[0].double(), 0).cpu() * n
    got = torch.bincount(out.cpu().long(), minlength=50)
    assert bool(((got - want).abs() <= 1.0).all())


def test_graph_and_stream(torch, hip):
    """Captured once, replayed on new logits with eager work between."""
    x, u = logits_like(torch, 4, 32000, "bfloat16"), uniform(torch, 4).cuda()
    p = torch.full((4,), 0.9, device="cuda")
    out, ws = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(hip.sample_workspace(x), dtype=torch.uint8, device="cuda")
    hip.sample(x, u, out, top_p=p, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.sample(x, u, out, top_p=p, workspace=ws)
    for seed in range(4):
        x.copy_(logits_like(torch, 4, 32000, "bfloat16", seed))
        graph.replay()
        torch.cuda.synchronize()
        assert out.tolist() == reference(torch, x, u, p=p)[0]
        eager = torch.empty_like(out)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            hip.sample(x, u, eager, top_p=p)
        side.synchronize()
        assert torch.equal(out, eager)


def test_agrees_with_argmax(torch, hip):
    """Temperature 0 is mh_argmax, which the decoder's greedy choice follows."""
    x = logits_like(torch, 9, 5000, "bfloat16")
    a, b = torch.empty(9, dtype=torch.int32, device="cuda"), torch.empty(9, dtype=torch.int32, device="cuda")
    hip.argmax(x, a, 9, 5000)
    hip.sample(x, uniform(torch, 9).cuda(), b, temperature=torch.zeros(9, device="cuda"))
    assert torch.equal(a, b)


def test_wrapper_refusals(torch, hip):
    x, u, out = torch.zeros((2, 8), device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, kw, match in (((x.double(), u, out), {}, "float32 or float16"), ((x, u[:1], out), {}, "u must be of shape"),
                            ((x, u, out.long()), {}, "int32"), ((x, u.double(), out), {}, "float32"),
                            ((x, u, out), dict(top_k=u), "int32"), ((x, u, out), dict(top_p=out), "float32"),
                            ((x.t().contiguous().t(), u, out), {}, "contiguous along a row"), ((x, u.cpu(), out), {}, "one GPU"),
                            ((x[0], u, out), {}, "shape"), ((x, u, out), dict(logprob=u.half()), "float32")):
        with pytest.raises(ValueError, match=match):
            hip.sample(*args, **kw)
