"""The paged 8-bit KV cache on the GPU: page plans and stored bits against exact
restatements, attention against the formula in 64 bits.

Tolerance of attention, per output: with A = sum_j w_j |v_j| / sum_j w_j of that
output and Q = the largest sum_d |q_d k_jd| scale over its keys,
  half a step of the output type times |o|            (the output's rounding)
+ 2^-11 A for 16-bit types, 2^-21 A for float32       (w in fp16: half a step is
                                                       2^-12 each, and the sum's; two
                                                       parts of 11 bits)
+ 2 (hd + 8) 2^-24 Q A                                (fp32 sums of scores, in w)
+ (n_keys / 16 + 64) 2^-24 A                          (fp32 sums over the keys: a lane
                                                       adds a sixteenth of them)
+ 2^-126 where all of these vanish.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E4M3_NAN = 0x7F


@pytest.fixture(scope="module")
def torch(hip):
    import torch as t
    return t


DTYPES = ["bfloat16", "float16", "float32"]
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}


# ---- plain statements ------------------------------------------------------------

def plan_reference(lens, new, free, tables, P, cap):
    """Integer arithmetic, one token at a time."""
    tables, slots, positions, cu, at, bad = [list(r) for r in tables], [], [], [0], 0, False
    width = len(tables[0]) if tables else 0
    for b, (n0, n1) in enumerate(zip(lens, new)):
        n0, n1 = max(n0, 0), max(n1, 0)
        for i in range(-(-n0 // P), min(-(-(n0 + n1) // P), width)):
            tables[b][i] = free[at] if at < len(free) else -1
            at += 1
        for t in range(n0, n0 + n1):
            page = tables[b][t // P] if t // P < width else -1
            if len(slots) < cap:
                slots.append(page * P + t % P if page >= 0 else -1)
                positions.append(t)
                bad |= page < 0
            else:
                bad = True
        cu.append(min(cu[-1] + n1, cap))
    pad = cap - len(slots)
    return {"tables": tables, "total": [max(a, 0) + max(b, 0) for a, b in zip(lens, new)], "cu": cu, "slots": slots + [-1] * pad,
            "positions": positions + [0] * pad, "used": [at], "bad": bad}


def e4m3_values(torch):
    """The value of each of the 256 bytes (float64, NaN for two)."""
    v = []
    for b in range(256):
        s, e, m = b >> 7, b >> 3 & 15, b & 7
        x = math.nan if e == 15 and m == 7 else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        v.append(-x if s else x)
    return torch.tensor(v, dtype=torch.float64)


def nearest_e4m3(torch, x):
    """Nearest e4m3 byte in 64 bits, ties to the even mantissa; not finite: NaN."""
    pos = e4m3_values(torch)[:127].numpy()  # 0 .. 448, increasing
    a = np.abs(x.numpy())
    ok = np.isfinite(a)
    a = np.where(ok, a, 0.0)
    hi = np.clip(np.searchsorted(pos, a), 0, 126)
    lo = np.clip(hi - 1, 0, 126)
    up, down = pos[hi] - a, a - pos[lo]
    q = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    q = np.where(ok, q, E4M3_NAN)
    return torch.from_numpy((q | np.where(ok & np.signbit(x.numpy()), 128, 0)).astype(np.uint8))


def least_scale(amax):
    if amax == 0:
        return 2.0 ** -100
    e = math.ceil(math.log2(amax / 448)) - 1
    while amax > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** max(e, -100)


def store_reference(torch, x, slots, cache, scale, P, transposed):
    """x [n, heads, hd] float64 into cache [pages, heads, P, hd] (uint8), runs of a page at a time."""
    cache = (cache.transpose(2, 3) if transposed else cache).contiguous().clone()
    scale, val, t = scale.double().clone(), e4m3_values(torch), 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and (slots[t] + n) % P:
            n += 1
        g, first = slots[t] // P, slots[t] % P
        for h in range(x.shape[1]):
            new = x[t:t + n, h]
            fin = new[torch.isfinite(new)]
            want = least_scale(float(fin.abs().max()) if fin.numel() else 0.0)
            now = want if first == 0 else max(want, float(scale[g, h]))
            if first and now > float(scale[g, h]):
                cache[g, h, :first] = nearest_e4m3(torch, val[cache[g, h, :first].long()] * (float(scale[g, h]) / now))
            cache[g, h, first:first + n] = nearest_e4m3(torch, new / now)
            scale[g, h] = now
        t += n
    return (cache.transpose(2, 3).contiguous() if transposed else cache), scale


def attend_reference(torch, c, q, out0, scale=None):
    """(outputs in float64, tolerance) for a Cache and its queries, one row at a time."""
    hd, G = q.shape[2], q.shape[1] // c.kv
    val = e4m3_values(torch)
    out = out0.double().cpu().clone()
    tol = torch.zeros_like(out)
    qd = q.double().cpu()
    scale = 1 / math.sqrt(hd) if scale is None else scale
    half = HALF_STEP[str(q.dtype).split(".")[1]]
    kc, vc, ks, vs = c.kc.cpu(), c.vc.cpu(), c.ks.double().cpu(), c.vs.double().cpu()
    for b, n_all in enumerate(c.lens):
        r0, r1 = c.cu[b], c.cu[b + 1]
        if r1 == r0:
            continue
        held = [(t, c.tables[b][t // c.P]) for t in range(min(n_all, len(c.tables[b]) * c.P))]
        tok = torch.tensor([t for t, p in held if 0 <= p < c.n_pages], dtype=torch.long)
        page = torch.tensor([p for t, p in held if 0 <= p < c.n_pages], dtype=torch.long)
        for h in range(c.kv):
            k = val[kc[page, h, tok % c.P].long()] * ks[page, h, None]
            v = val[vc[page, h, :, tok % c.P].long()] * vs[page, h, None]
            for i in range(r1 - r0):
                p = n_all - (r1 - r0) + i
                see = torch.ones(len(tok), dtype=torch.bool)
                if c.causal:
                    see &= tok <= p
                if c.window:
                    see &= tok > p - c.window
                rows = qd[r0 + i, h * G:(h + 1) * G]
                if not see.any():
                    out[r0 + i, h * G:(h + 1) * G] = 0
                    continue
                s = rows @ k[see].T * scale
                w = torch.exp(s - s.amax(1, keepdim=True))
                w = w / w.sum(1, keepdim=True)
                o = w @ v[see]
                out[r0 + i, h * G:(h + 1) * G] = o
                A, Q = w @ v[see].abs(), ((rows.abs() @ k[see].abs().T) * abs(scale)).amax(1, keepdim=True)
                tol[r0 + i, h * G:(h + 1) * G] = (
                    half * o.abs() + A * ((2.0 ** -11 if half > 2.0 ** -20 else 2.0 ** -21) + 2 * (hd + 8) * 2.0 ** -24 * Q
                                          + (int(see.sum()) / 16 + 64) * 2.0 ** -24) + 2.0 ** -126)
    return out, tol


def assert_within(torch, got, ref, tol, what=""):
    got = got.double().cpu()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places ({int(torch.isnan(got).sum())} against {int(nan.sum())})"
    off = torch.where(nan, 0.0, (got - ref).abs() - tol.nan_to_num(0.0))
    worst = int(off.argmax())
    assert float(off.max()) <= 0, f"{what}: {float(got.flatten()[worst])} against {float(ref.flatten()[worst])} +- {float(tol.flatten()[worst])}"


class Cache:
    """A pool with random contents for requests of the given lengths, `new` of each being queries."""

    def __init__(self, torch, kv, hd, P, lens, new, seed=0, causal=True, window=0, spare=3, spread=4.0, junk=True):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.hd, self.P, self.lens, self.causal, self.window = kv, hd, P, list(lens), causal, window
        need = [-(-n // P) for n in lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g).tolist()
        width, at, self.tables = max([1] + need), 0, []
        for k in need:
            self.tables.append(order[at:at + k] + [-1] * (width - k))
            at += k
        self.cu = [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        x = torch.randn((2, self.n_pages, kv, P, hd), generator=g) * 100
        b = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        if junk:  # what lies behind a request's last token, and in pages of nobody, is anything
            used = torch.zeros((self.n_pages, P), dtype=torch.bool)
            for n, row in zip(lens, self.tables):
                for t in range(n):
                    used[row[t // P], t % P] = True
            b = torch.where(used[None, :, None, :, None], b, torch.tensor(E4M3_NAN, dtype=torch.uint8))
        self.kc, self.vc = b[0].contiguous().cuda(), b[1].transpose(2, 3).contiguous().cuda()
        self.ks = (2.0 ** torch.randint(-9, -6, (self.n_pages, kv), generator=g)).float().cuda()
        self.vs = (2.0 ** torch.randint(-9, int(-9 + spread), (self.n_pages, kv), generator=g)).float().cuda()
        self.max_q, self.max_len = max(new), max(list(lens) + [0])
        self.sync(torch)

    def sync(self, torch):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.d_tables, self.d_lens, self.d_cu = i32(self.tables), i32(self.lens), i32(self.cu)

    def attend(self, hip, q, out, max_q=None, max_len=None, **kw):
        hip.attention_paged(q, self.kc, self.vc, self.ks, self.vs, self.d_tables, self.d_lens, self.d_cu, out,
                            self.max_q if max_q is None else max_q, self.max_len if max_len is None else max_len,
                            causal=self.causal, window=self.window, **kw)
        return out


def queries(torch, n, heads, hd, dtype, seed=1):
    return torch.randn((n, heads, hd), generator=torch.Generator().manual_seed(seed)).to(getattr(torch, dtype)).cuda()


def check(torch, hip, c, heads, dtype, seed=1, what="", extra=0, **kw):
    q = queries(torch, c.cu[-1] + extra, heads, c.hd, dtype, seed)
    out = torch.full_like(q, 7.0)
    print(f"attention_paged {what} {dtype} heads {heads}/{c.kv} hd {c.hd} page {c.P} lens {c.lens[:6]} cu {c.cu[:6]}", flush=True)
    ref, tol = attend_reference(torch, c, q, out, kw.get("scale"))
    c.attend(hip, q, out, **kw)
    torch.cuda.synchronize()
    assert_within(torch, out, ref, tol, what)
    return out


# ---- page_plan ---------------------------------------------------------------------

@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("lens,new,n_free,width,cap", [
    ([0], [1], 4, 4, 1), ([15, 16, 17, 0], [1, 1, 1, 1], 9, 3, 4), ([0, 5, 300, 31], [700, 0, 1, 33], 70, 50, 740),
    ([3] * 300, [1] * 300, 0, 1, 300), ([64] * 300, [2] * 300, 400, 6, 700), ([0, 0], [0, 0], 0, 0, 3),
    ([-4, 10], [5, -6], 2, 2, 8),                       # negative counts are none
    ([77], [20000], 1300, 1400, 30000), ([9, 0, 40], [1, 9000, 2000], 700, 600, 11500),  # several workgroups to a request
    ([0, 0, 0], [100, 100, 100], 5, 20, 300),           # free pages end
    ([10, 10], [400, 20], 60, 2, 500),                  # the table's width ends
    ([0, 0], [30, 30], 9, 9, 41)])                      # the slots end
def test_page_plan(torch, hip, P, lens, new, n_free, width, cap):
    rng = np.random.default_rng(P + len(lens))
    n_pages = 3000
    pages = rng.permutation(n_pages).tolist()
    free, rest = pages[:n_free], pages[n_free:]
    tables = [[rest.pop() if i < -(-max(n, 0) // P) else -1 for i in range(width)] for n in lens]
    want = plan_reference(lens, new, free, tables, P, cap)
    i32 = lambda v, shape=None: torch.tensor(v, dtype=torch.int32, device="cuda").reshape(shape or (len(v),))  # noqa: E731
    d_tables, fill = i32(tables, (len(lens), width)), lambda n: torch.full((n,), 99, dtype=torch.int32, device="cuda")  # noqa: E731
    total, cu, slots, positions, used = fill(len(lens)), fill(len(lens) + 1), fill(cap), fill(cap), fill(1)
    hip.check_device_errors()
    hip.page_plan(i32(lens), i32(new), i32(free), d_tables, total, cu, slots, positions, used, P, n_pages)
    got = {"tables": d_tables.tolist(), "total": total.tolist(), "cu": cu.tolist(), "slots": slots.tolist(),
           "positions": positions.tolist(), "used": used.tolist()}
    for k in got:
        assert got[k] == want[k], k
    if want["bad"]:
        from munet_amd._lib import HipError
        with pytest.raises(HipError, match="page_plan"):
            hip.check_device_errors()
    hip.check_device_errors()


def test_page_plan_refuses_pages_outside_the_pool(torch, hip):
    from munet_amd._lib import HipError
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tables, out = i32([[5, -1], [900, -1]]), [i32([0] * n) for n in (2, 3, 40, 1)]
    hip.page_plan(i32([4, 4]), i32([20, 20]), i32([6, 77]), tables, out[0], out[1], out[2], None, out[3], 16, 50)
    assert tables.tolist() == [[5, 6], [900, -1]]
    assert out[2].tolist() == [84 + i for i in range(12)] + [96 + i for i in range(8)] + [-1] * 20
    with pytest.raises(HipError, match="page_plan"):
        hip.check_device_errors()


# ---- kv_store_paged ------------------------------------------------------------------

def _store(torch, hip, x, slots, cache, scales, P):
    kc, vc = cache[0].cuda().clone(), cache[1].transpose(2, 3).contiguous().cuda()
    ks, vs = scales[0].cuda().clone(), scales[1].cuda().clone()
    sl = torch.tensor(slots, dtype=torch.int32, device="cuda")
    hip.kv_store_paged(x[0], x[1], sl, kc, vc, ks, vs)
    torch.cuda.synchronize()
    wk, sk = store_reference(torch, x[0].double().cpu(), slots, cache[0], scales[0], P, False)
    wv, sv = store_reference(torch, x[1].double().cpu(), slots, cache[1].transpose(2, 3), scales[1], P, True)
    assert torch.equal(ks.double().cpu(), sk) and torch.equal(vs.double().cpu(), sv)
    nan = lambda b: torch.where(b.bitwise_and(127) == 127, 127, b)  # (a NaN's sign is not specified)  # noqa: E731
    assert torch.equal(nan(kc.cpu()), nan(wk)), "keys"
    assert torch.equal(nan(vc.cpu()), nan(wv)), "values"
    return kc, vc, ks, vs


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("P,kv,hd,runs", [
    (16, 1, 16, [(2, 0, 1)]), (16, 3, 64, [(0, 15, 1), (5, 0, 16), (3, 4, 9)]), (64, 2, 128, [(1, 63, 1), (2, 0, 64), (4, 0, 7), (0, 5, 1)]),
    (32, 12, 64, [(7, 31, 1), (3, 30, 2)]), (128, 2, 80, [(0, 17, 100), (1, 0, 128), (6, 127, 1)]),
    (256, 1, 256, [(2, 100, 156), (3, 0, 200), (5, 255, 1)]), (16, 40, 32, [(i, i % 16, 1) for i in range(8)])])
def test_kv_store(torch, hip, dtype, P, kv, hd, runs):
    """(page, place, tokens) runs: fresh pages, pages appended to with and without a larger scale, rows inside a wider row."""
    g = torch.Generator().manual_seed(P * 7 + hd)
    slots = []
    for page, place, n in runs:
        slots += [page * P + place + i for i in range(n)] + [-1]
    rows = torch.randn((len(slots), 2, kv, hd), generator=g)
    rows *= torch.exp2(torch.randint(-3, 4, (len(slots), 1, 1, 1), generator=g).float())
    rows = rows.to(getattr(torch, dtype)).cuda()
    cache = [torch.randn((8, kv, P, hd), generator=g).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-12, -2, (8, kv), generator=g).float()) for _ in range(2)]
    print(f"kv_store {dtype} P {P} kv {kv} hd {hd}", flush=True)
    _store(torch, hip, (rows[:, 0], rows[:, 1]), slots, cache, scales, P)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("P,hd", [(64, 128), (128, 128), (128, 80), (256, 64), (256, 128), (256, 256), (64, 256)])
def test_kv_store_prompts(torch, hip, dtype, P, hd):
    """Tokens enough for workgroups that look after several: whole pages, and parts of pages behind and before others."""
    g, kv = torch.Generator().manual_seed(P + hd), 8
    runs, pages = [(1, P - 3, 3), (2, 5, P // 2), (3, P // 4 + 1, 2)], 24
    runs += [(p, 0, P) for p in range(4, 4 + 1024 // P)] + [(20, 0, P - 1), (21, 0, 1), (22, 13, P - 13)]
    slots = []
    for page, place, n in runs:
        slots += [page * P + place + i for i in range(n)]
    assert len(slots) * kv >= 8192
    rows = torch.randn((len(slots), 2, kv, hd), generator=g)
    rows *= torch.exp2(torch.randint(-3, 4, (len(slots), 1, 1, 1), generator=g).float())
    rows = rows.to(getattr(torch, dtype)).cuda()
    cache = [torch.randn((pages, kv, P, hd), generator=g).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-12, -2, (pages, kv), generator=g).float()) for _ in range(2)]
    print(f"kv_store prompts {dtype} P {P} hd {hd}", flush=True)
    _store(torch, hip, (rows[:, 0], rows[:, 1]), slots, cache, scales, P)


def test_kv_store_rounds_every_value(torch, hip):
    """All fp16 values: ties, subnormals of e4m3, NaN and infinities, and each magnitude as its own page's largest."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = bits.reshape(4096, 1, 16).cuda()
    cache = [torch.zeros((256, 1, 16, 16), dtype=torch.uint8) for _ in range(2)]
    scales = [torch.ones((256, 1)) for _ in range(2)]
    _store(torch, hip, (x, x), list(range(4096)), cache, scales, 16)
    one = torch.arange(1, 0x7F800000, 8388608 // 8 + 1, dtype=torch.int64).to(torch.int32).view(torch.float32)  # every binade, 8 each
    n = one.numel()
    x = torch.zeros((n, 1, 16))
    x[:, 0, 3] = one
    x[:, 0, 5] = -one / 3
    cache = [torch.zeros((n, 1, 16, 16), dtype=torch.uint8) for _ in range(2)]
    _store(torch, hip, (x.cuda(), x.cuda()), [16 * i for i in range(n)], cache, [torch.ones((n, 1)) for _ in range(2)], 16)


def test_kv_store_slots_outside_the_pool(torch, hip):
    from munet_amd._lib import HipError
    x = torch.ones((4, 1, 16), device="cuda")
    kc, vc = torch.zeros((3, 1, 16, 16), dtype=torch.uint8, device="cuda"), torch.zeros((3, 1, 16, 16), dtype=torch.uint8, device="cuda")
    ks, vs = torch.ones((3, 1), device="cuda"), torch.ones((3, 1), device="cuda")
    hip.kv_store_paged(x, x, torch.tensor([-7, 48, 2 ** 31 - 1, 33], dtype=torch.int32, device="cuda"), kc, vc, ks, vs)
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()
    assert int((kc != 0).sum()) == 16 and int((vc != 0).sum()) == 16 and bool((kc[2, 0, 1] != 0).all()) and bool((vc[2, 0, :, 1] != 0).all())


# ---- attention_paged --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,hd", [(1, 1, 64), (12, 12, 64), (8, 2, 128), (5, 1, 32), (16, 1, 80), (34, 2, 16), (4, 2, 256), (6, 2, 176)])
@pytest.mark.parametrize("P", [16, 64, 256])
def test_decode(torch, hip, dtype, heads, kv, hd, P):
    lens = [1, 16, 63, 64, 65, 257, 0, 130]
    check(torch, hip, Cache(torch, kv, hd, P, lens, [1] * len(lens), seed=hd + P), heads, dtype, what="decode")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,hd,P", [(2, 2, 64, 16), (8, 2, 128, 64), (3, 1, 96, 32), (4, 4, 256, 128)])
@pytest.mark.parametrize("window", [0, 1, 40])
def test_prompts_and_chunks(torch, hip, dtype, heads, kv, hd, P, window):
    """Whole prompts, chunks behind a prefix, single tokens and none at all in one batch, with rows of no request behind."""
    lens, new = [70, 1, 200, 33, 64, 90], [70, 1, 9, 33, 0, 65]
    out = check(torch, hip, Cache(torch, kv, hd, P, lens, new, seed=hd, window=window), heads, dtype, what="prompts", extra=5)
    assert bool((out[-5:] == 7.0).all())


@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_not_causal(torch, hip, dtype, window):
    check(torch, hip, Cache(torch, 2, 64, 32, [50, 130, 7], [50, 20, 3], causal=False, window=window), 4, dtype, what="not causal")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,hd,new", [(4, 4, 64, 1), (8, 1, 128, 3), (2, 1, 256, 1), (8, 2, 64, 40)])
def test_keys_split_over_workgroups(torch, hip, dtype, heads, kv, hd, new):
    """Long requests beside short ones: several shares of the keys, most of them empty for the short."""
    c = Cache(torch, kv, hd, 64, [3000, new, 700], [new, new, new], seed=3)
    q = queries(torch, c.cu[-1], heads, hd, dtype)
    assert hip.attention_paged_workspace(q, c.kc, c.d_lens, c.max_q, c.max_len) > 0
    check(torch, hip, c, heads, dtype, what="split")


def test_bounds_lower_than_the_lengths(torch, hip):
    """max_q and max_len only size the launch."""
    c = Cache(torch, 2, 64, 16, [900, 300, 50], [5, 290, 50], seed=5)
    check(torch, hip, c, 4, "bfloat16", what="low bounds", max_q=1, max_len=300)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scale_and_more_queries_than_keys(torch, hip, dtype):
    """Queries before position 0 see nothing."""
    check(torch, hip, Cache(torch, 1, 64, 16, [3, 20], [9, 20]), 2, dtype, what="scale", scale=0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 30])
def test_not_a_number_reaches_only_who_sees_it(torch, hip, dtype, new):
    """A NaN key or value: NaN for the queries that see it, nothing for those before it or past the window."""
    for what in ("key", "value"):
        c = Cache(torch, 1, 64, 16, [100, 41], [new, min(new, 41)], seed=9, window=25)
        for t in (60, 85, 99):
            page, place = c.tables[0][t // 16], t % 16
            if what == "key":
                c.kc[page, 0, place, 7] = E4M3_NAN
            else:
                c.vc[page, 0, 5, place] = 0xFF
        out = check(torch, hip, c, 2, dtype, what=f"NaN {what}")
        assert bool(torch.isnan(out).any()) and not bool(torch.isnan(out[c.cu[1]:]).any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_and_large_queries_stay_in_their_rows(torch, hip, dtype):
    c = Cache(torch, 1, 64, 16, [50], [20])
    q = queries(torch, 20, 2, 64, dtype)
    plain = c.attend(hip, q, torch.empty_like(q)).clone()
    q2 = q.clone()
    q2[3, 0, 0] = math.inf
    q2[4, 1, 3] = math.nan
    q2[5, 0] = 0
    q2[6, 1] = min(torch.finfo(q.dtype).max / 4, 2.0 ** 60)
    q2[7, 0] *= 2.0 ** -20
    out = c.attend(hip, q2, torch.empty_like(q))
    same = torch.ones((20, 2), dtype=torch.bool)
    for r, h in ((3, 0), (4, 1), (5, 0), (6, 1), (7, 0)):
        same[r, h] = False
    assert torch.equal(out.cpu()[same], plain.cpu()[same])
    assert bool(torch.isnan(out[4, 1]).all())
    q2[3, 0, 0] = 1.0
    q2[4, 1, 3] = 1.0
    ref, tol = attend_reference(torch, c, q2, out)
    out = c.attend(hip, q2, torch.empty_like(q))
    keep = torch.ones((20, 2), dtype=torch.bool)
    keep[6, 1] = False  # (scores of 10^30: the largest alone counts, and its fp32 rounding decides which)
    assert_within(torch, out.cpu()[keep], ref[keep], tol[keep], "large and small rows")
    assert bool(torch.isfinite(out[6, 1]).all())


@pytest.mark.parametrize("spread", [4.0, 60.0])
def test_value_scales_far_apart(torch, hip, spread):
    """Pages whose value scales differ by up to 2^60: the largest decides, to its precision."""
    check(torch, hip, Cache(torch, 2, 64, 16, [200, 90], [1, 30], spread=spread, seed=4), 4, "bfloat16", what="value scales")


@pytest.mark.parametrize("P", [32, 64, 128])
@pytest.mark.parametrize("dtype,hd", [("bfloat16", 128), ("float32", 64), ("float16", 256)])
def test_prompts_over_pages_outside_the_pool(torch, hip, P, dtype, hd):
    """Prompts whose blocks lie in one page each and in several, some pages missing, scales far apart."""
    from munet_amd._lib import HipError
    c = Cache(torch, 2, hd, P, [700, 333, 64], [200, 333, 40], spread=4.0 if dtype == "float16" else 40.0, seed=P)
    c.tables[0][2], c.tables[0][-1], c.tables[1][0] = -1, c.n_pages + 5, 2 ** 31 - 1
    c.sync(torch)
    hip.check_device_errors()
    check(torch, hip, c, 4, dtype, what="prompts, bad pages")
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()


def test_pages_outside_the_pool_hold_no_keys(torch, hip):
    from munet_amd._lib import HipError
    c = Cache(torch, 2, 64, 16, [100, 40], [1, 30], seed=6)
    c.tables[0][2], c.tables[1][1] = -1, c.n_pages + 5
    c.sync(torch)
    check(torch, hip, c, 4, "bfloat16", what="bad pages")
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()
    c = Cache(torch, 2, 64, 16, [100, 40], [1, 1], seed=6)
    c.d_lens = torch.tensor([2 ** 31 - 1, 40], dtype=torch.int32, device="cuda")  # past the table: cut
    q = queries(torch, 2, 4, 64, "bfloat16")
    out = c.attend(hip, q, torch.empty_like(q))
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()
    c.lens = [112, 40]
    c.sync(torch)
    c2 = c.attend(hip, q, torch.empty_like(q))
    assert torch.equal(out[1], c2[1])


def test_pool_beyond_32_bits(torch, hip):
    """A request in the last pages of a pool of 5 GiB a cache."""
    kv, hd, P = 8, 128, 64
    n_pages = 5 * (1 << 30) // (kv * hd * P)
    c = Cache(torch, kv, hd, P, [150, 70], [1, 70], seed=8, spare=0)
    n = c.n_pages
    for name in ("kc", "vc"):
        small = getattr(c, name)
        big = torch.zeros((n_pages,) + tuple(small.shape[1:]), dtype=torch.uint8, device="cuda")
        big[-n:] = small
        setattr(c, name, big)
    for name in ("ks", "vs"):
        setattr(c, name, torch.cat([torch.ones((n_pages - n, kv), device="cuda"), getattr(c, name)]))
    q = queries(torch, 71, 16, hd, "bfloat16")
    far = torch.tensor([[p + n_pages - n if p >= 0 else -1 for p in row] for row in c.tables], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    hip.attention_paged(q, c.kc, c.vc, c.ks, c.vs, far, c.d_lens, c.d_cu, out, 70, 150)
    for name in ("kc", "vc", "ks", "vs"):
        setattr(c, name, getattr(c, name)[-n:].contiguous())
    near = c.attend(hip, q, torch.empty_like(q))
    assert torch.equal(out, near)
    x = torch.randn((3, 2, kv, hd), device="cuda")
    big = [torch.zeros((n_pages,) + s, dtype=torch.uint8, device="cuda") for s in ((kv, P, hd), (kv, hd, P))]
    sc = [torch.ones((n_pages, kv), device="cuda") for _ in range(2)]
    last = (n_pages - 1) * P
    hip.kv_store_paged(x[:, 0], x[:, 1], torch.tensor([last, last + 1, last + 2], dtype=torch.int32, device="cuda"), *big, *sc)
    assert int((big[0][:-1] != 0).sum()) == 0 and bool((big[0][-1, :, :3].float().abs().sum(-1) > 0).all())
    assert bool((big[1][-1, :, :, :3].float().abs().sum(-2) > 0).all()) and int((big[1][-1, :, :, 3:] != 0).sum()) == 0


def test_rows_inside_wider_rows(torch, hip):
    """q and out as slices of a fused projection's rows, out of another width."""
    c = Cache(torch, 2, 64, 16, [40, 9], [20, 9])
    wide = queries(torch, 29, 12, 64, "float16")
    q, out = wide[:, 2:6], torch.zeros((29, 9, 64), dtype=torch.float16, device="cuda")
    c.attend(hip, q, out[:, 1:5])
    assert torch.equal(out[:, 1:5], c.attend(hip, q.contiguous(), torch.empty_like(q.contiguous())))
    assert not bool(out[:, 0].any()) and not bool(out[:, 5:].any())


def test_a_step_together(torch, hip):
    """plan, store, attend for prompts, then for single tokens: what the cache gives equals attention over its own values,
    and those are the stored ones within an e4m3 half step."""
    kv, hd, P, heads, n_pages, width = 2, 64, 16, 4, 40, 8
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tables, lens, free = torch.full((3, width), -1, dtype=torch.int32, device="cuda"), i32([0, 0, 0]), list(range(n_pages))[::-1]
    kc, vc = torch.zeros((n_pages, kv, P, hd), dtype=torch.uint8, device="cuda"), torch.zeros((n_pages, kv, hd, P), dtype=torch.uint8, device="cuda")
    ks, vs = torch.zeros((n_pages, kv), device="cuda"), torch.zeros((n_pages, kv), device="cuda")
    held = [[], [], []]
    for step, new in enumerate(([37, 16, 5], [1, 1, 1], [1, 0, 1], [30, 1, 20])):
        n = sum(new)
        total, cu, slots, pos, used = i32([0] * 3), i32([0] * 4), i32([0] * (n + 3)), i32([0] * (n + 3)), i32([0])
        hip.page_plan(lens, i32(new), i32(free), tables, total, cu, slots, pos, used, P, n_pages)
        free = free[int(used):]
        rows = queries(torch, n + 3, heads + 2 * kv, hd, "bfloat16", seed=step)
        q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
        hip.kv_store_paged(k, v, slots, kc, vc, ks, vs)
        out = torch.full((n + 3, heads, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        hip.attention_paged(q, kc, vc, ks, vs, tables, total, cu, out, max(new), int(total.max()))
        hip.check_device_errors()
        at = 0
        for b in range(3):
            held[b].append(k[at:at + new[b]].float())
            at += new[b]
        c = Cache.__new__(Cache)
        c.kv, c.hd, c.P, c.n_pages, c.causal, c.window = kv, hd, P, n_pages, True, 0
        c.kc, c.vc, c.ks, c.vs = kc, vc, ks, vs
        c.lens, c.cu, c.tables = total.tolist(), cu.tolist(), tables.tolist()
        ref, tol = attend_reference(torch, c, q, torch.full_like(out, 7.0))
        assert_within(torch, out, ref, tol, f"step {step}")
        for b in range(3):
            want = torch.cat(held[b])
            t = torch.arange(len(want), device="cuda")
            page = tables[b].long()[t // P]
            got = kc.view(torch.float8_e4m3fn).float()[page, :, t % P] * ks[page][..., None]
            # half a step of the value, or of the smallest values (2^-10 of the scale), once for each of at most two roundings
            bound = torch.maximum(want.abs() * 2.0 ** -4, ks[page][..., None] * 2.0 ** -10) * 2
            assert bool(((got - want).abs() <= bound).all())
        lens = total


def test_graph_and_streams(torch, hip):
    """A step captured once and replayed on new lengths, with eager work between, each replay against the eager result;
    two captured calls with a workspace each; a call on another stream."""
    kv, hd, P, heads, B = 2, 64, 16, 4, 3
    lens0 = [700, 33, 300]
    c = Cache(torch, kv, hd, P, lens0, [1] * B, seed=11, junk=False)
    n_pages = c.n_pages
    q = queries(torch, B, heads, hd, "bfloat16")
    k = queries(torch, B, kv, hd, "bfloat16", seed=2)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, one, free = i32([n - 1 for n in lens0]), i32([1] * B), i32([])
    bufs = [i32([0] * n) for n in (B, B + 1, B, B, 1)]
    out = torch.empty_like(q)
    ws = torch.empty(hip.attention_paged_workspace(q, c.kc, c.d_lens, 1, 700), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0

    def step(o, w):
        hip.page_plan(lens, one, free, c.d_tables, bufs[0], bufs[1], bufs[2], bufs[3], bufs[4], P, n_pages)
        hip.kv_store_paged(k, k, bufs[2], c.kc, c.vc, c.ks, c.vs)
        hip.attention_paged(q, c.kc, c.vc, c.ks, c.vs, c.d_tables, bufs[0], bufs[1], o, 1, 700, workspace=w)

    step(out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, ws)
    out2, ws2 = torch.empty_like(q), torch.empty_like(ws)
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        hip.attention_paged(q, c.kc, c.vc, c.ks, c.vs, c.d_tables, bufs[0], bufs[1], out2, 1, 700, workspace=ws2)
    for at in ([699, 32, 299], [100, 5, 200], [640, 0, 31], [699, 32, 299]):
        lens.copy_(i32(at))
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        got, got2 = out.clone(), out2.clone()
        eager = torch.empty_like(q)
        step(eager, torch.empty_like(ws))
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(got2, eager), at
    side, o3 = torch.cuda.Stream(), torch.empty_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.d_lens, c.d_cu = bufs[0], bufs[1]
        c.attend(hip, q, o3)
    side.synchronize()
    assert torch.equal(o3, eager)


def test_repeated_calls_give_the_same_bits(torch, hip):
    c = Cache(torch, 2, 128, 64, [3000, 500], [1, 1])
    q = queries(torch, 2, 8, 128, "bfloat16")
    first = c.attend(hip, q, torch.empty_like(q))
    for _ in range(3):
        assert torch.equal(first, c.attend(hip, q, torch.empty_like(q)))


def test_wrapper_refusals(torch, hip):
    c = Cache(torch, 2, 64, 16, [40], [1])
    q = queries(torch, 1, 4, 64, "bfloat16")
    out = torch.empty_like(q)
    base = dict(q=q, k_cache=c.kc, v_cache=c.vc, k_scale=c.ks, v_scale=c.vs, tables=c.d_tables, lens=c.d_lens, cu=c.d_cu, out=out,
                max_q=1, max_len=40)
    for change, match in ((dict(v_cache=c.kc), "v_cache must be of shape"), (dict(q=q.double()), "float32 or float16"),
                          (dict(out=out.float()), "out must be bfloat16"), (dict(tables=c.d_tables.long()), "int32"),
                          (dict(k_scale=c.ks.half()), "float32"), (dict(cu=c.d_cu[:1]), "shape"), (dict(lens=c.d_lens.cpu()), "one GPU"),
                          (dict(q=q.transpose(1, 2)), "shape"), (dict(k_cache=c.kc.float()), "uint8"), (dict(scale=0.0), "scale 0"),
                          (dict(q=torch.empty((1, 64, 4), dtype=q.dtype, device="cuda").transpose(1, 2)), "contiguous")):
        with pytest.raises(ValueError, match=match):
            hip.attention_paged(**{**base, **change})
    with pytest.raises(ValueError, match="v must be bfloat16"):
        hip.kv_store_paged(q[:, :2], q[:, :2].float(), c.d_lens, c.kc, c.vc, c.ks, c.vs)
    with pytest.raises(ValueError, match="slots must be of shape"):
        hip.kv_store_paged(q[:, :2], q[:, :2], c.d_cu, c.kc, c.vc, c.ks, c.vs)
