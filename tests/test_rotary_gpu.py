"""Rotary positions on the GPU: tables and rotations against the formulas in 64
bits, rotated appends against the same keys stored by the call without rotation.

Tolerances.  A table's value v = m cos a or m sin a: half a step of float32
(2^-24 |v|), and the angle's error: position, frequency and their product round to
64 bits, the angle is reduced with one more rounding of each, 8 2^-53 |a| m in all.
A rotated value a c - b s: one rounding of a product and one of the sum in
float32, 2^-24 (|a c| + |b s|) each, then half a step of the output type; 2^-25
where fp16 has no smaller step (2^-149 for the others)."""
import numpy as np
import pytest

from test_paged_gpu import DTYPES, HALF_STEP, e4m3_values

pytestmark = pytest.mark.gpu

LEAST = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25, "float32": 2.0 ** -149}


@pytest.fixture(scope="module")
def torch(hip):
    import torch as t
    from munet_amd._lib import HipError
    try:  # (errors that tests of other files left set)
        hip.check_device_errors()
    except HipError:
        pass
    return t


def normal(torch, seed, shape, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(getattr(torch, dtype)).cuda()


def table_of(torch, seed, n, half):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand((n, half), generator=g, dtype=torch.float64) * 6.4
    return torch.stack([a.cos(), a.sin()], -1).float().cuda()


# ---- tables --------------------------------------------------------------------------

@pytest.mark.parametrize("n,rot", [(1, 2), (1, 128), (5, 24), (64, 64), (333, 130), (4099, 128)])
@pytest.mark.parametrize("scaling", [None, "turns"])
def test_table(hip, torch, n, rot, scaling):
    from munet_amd.backend import rotary_frequencies
    freq, m = rotary_frequencies(rot, 10000.0, scaling, 8.0, 4096)
    rng = np.random.default_rng(n + rot)
    pos = rng.integers(0, 131072, n).astype(np.int32)
    # the ends of int32, the places next to zero, and whole turns of the first pair
    ends = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 710, 103993, 1146408], np.int32)
    pos[:min(n, 8)] = ends[:n]
    got = torch.full((n + 1, rot // 2, 2), 7.0, device="cuda")
    hip.rotary_table(torch.from_numpy(pos).cuda(), torch.from_numpy(freq).cuda(), got[:n], magnitude=m)
    a = pos.astype(np.float64)[:, None] * freq
    want = np.stack([np.cos(a), np.sin(a)], -1) * m
    tol = 2.0 ** -24 * np.abs(want) + 8 * 2.0 ** -53 * np.abs(a)[..., None] * m + 2.0 ** -50
    off = np.abs(got[:n].double().cpu().numpy() - want)
    assert (off <= tol).all(), np.argwhere(off > tol)[:4]
    assert (got[n] == 7.0).all()


# ---- rotations -----------------------------------------------------------------------

def rotation(x, table, interleaved, inverse=False):
    """The formula in 64 bits and what its roundings in float32 may add."""
    x, t = x.double().cpu().numpy(), table.double().cpu().numpy()
    h = t.shape[1]
    c, s = t[:, None, :, 0], t[:, None, :, 1] * (-1.0 if inverse else 1.0)
    ia = slice(0, 2 * h, 2) if interleaved else slice(0, h)
    ib = slice(1, 2 * h, 2) if interleaved else slice(h, 2 * h)
    y, err = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    err[..., ia] = 2 * 2.0 ** -24 * (np.abs(a * c) + np.abs(b * s))
    err[..., ib] = 2 * 2.0 ** -24 * (np.abs(a * s) + np.abs(b * c))
    return y, err


def check(got, y, err, dtype):
    off = np.abs(got.double().cpu().numpy() - y)
    bad = off > err + HALF_STEP[dtype] * (np.abs(y) + err) + LEAST[dtype]
    assert not bad.any(), (int(bad.sum()), off[bad].max())


SIZES = [(1, 1, 2, 2), (1, 24, 64, 64), (3, 5, 64, 24), (7, 2, 80, 40), (33, 3, 128, 128), (2, 7, 96, 34), (1100, 4, 128, 64), (5, 3, 7, 4),
         (65, 40, 128, 128), (4, 1, 256, 256), (9, 9, 48, 48), (17, 33, 32, 16), (2, 300, 64, 64), (3, 2, 33, 32),
         (70, 40, 128, 120), (9, 5, 128, 100), (1030, 11, 96, 42), (6, 2, 36, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,hd,rot", SIZES)
def test_rotary(hip, torch, dtype, interleaved, n, heads, hd, rot):
    x, table = normal(torch, n + hd, (n, heads, hd), dtype), table_of(torch, n, n, rot // 2)
    guard = torch.full((n + 1, heads, hd), 3.0, dtype=x.dtype, device="cuda")
    out = guard[:n]
    hip.rotary(x, table, out, interleaved=interleaved)
    check(out, *rotation(x, table, interleaved), dtype)
    assert torch.equal(out[..., rot:], x[..., rot:]) and (guard[n] == 3.0).all()
    back = torch.empty_like(x)
    hip.rotary(x, table, back, interleaved=interleaved, inverse=True)
    check(back, *rotation(x, table, interleaved, True), dtype)
    # in place, the same bits
    y = x.clone()
    hip.rotary(y, table, y, interleaved=interleaved)
    assert torch.equal(y, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("behind,first,width", [(2, 0, 64), (1, 1, 64), (3, 2, 65)])
def test_rotary_of_views(hip, torch, dtype, interleaved, behind, first, width):
    """Heads inside wider rows, read and written there; what lies beside them stays.
    Rows that start off 16 bytes too."""
    n, heads, hd = 21, 3, width
    wide = normal(torch, 3, (n, heads + behind, hd), dtype)
    table, before = table_of(torch, 4, n, 24), wide.clone()
    x = wide[:, first:first + heads]
    y, err = rotation(x, table, interleaved)
    other = torch.zeros((n, heads + 2, hd), dtype=wide.dtype, device="cuda")
    hip.rotary(x, table, other[:, 1:1 + heads], interleaved=interleaved)
    check(other[:, 1:1 + heads], y, err, dtype)
    assert not other[:, 0].any() and not other[:, -1].any() and torch.equal(wide, before)
    hip.rotary(x, table, x, interleaved=interleaved)
    check(x, y, err, dtype)
    beside = torch.ones(heads + behind, dtype=torch.bool)
    beside[first:first + heads] = False
    assert torch.equal(wide[:, beside], before[:, beside])


def test_rotary_between_columns_of_one_buffer(hip, torch):
    """Queries of a row rotated into other heads of the same rows; heads that meet are refused."""
    from munet_amd._lib import HipError
    wide = normal(torch, 5, (30, 8, 32), "float16")
    table, x = table_of(torch, 6, 30, 16), wide[:, :3].clone()
    hip.rotary(wide[:, :3], table, wide[:, 5:])
    check(wide[:, 5:], *rotation(x, table, False), "float16")
    assert torch.equal(wide[:, :3], x)
    with pytest.raises(HipError, match="overlaps"):
        hip.rotary(wide[:, :3], table, wide[:, 2:5])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_extremes(hip, torch, dtype):
    """NaN and infinities reach their own pair alone; the smallest values keep their steps."""
    x = normal(torch, 7, (4, 2, 64), dtype)
    x[0, 0, 3], x[1, 1, 40], x[2, 0, 0] = float("nan"), float("inf"), float("-inf")
    x[3] = torch.arange(128, device="cuda").reshape(2, 64).to(x.dtype) * torch.finfo(x.dtype).smallest_normal / 64
    table = table_of(torch, 8, 4, 32)
    out = torch.empty_like(x)
    hip.rotary(x, table, out)
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[0, 0, [3, 35]] = want[1, 1, [8, 40]] = want[2, 0, [0, 32]] = True
    assert torch.equal(bad, want)
    assert out[0, 0, 3].isnan() and out[0, 0, 35].isnan()
    check(out[3:], *rotation(x[3:], table[3:], False), dtype)


def test_gradient_is_the_inverse(hip, torch):
    """sum(g * rotary(x)) differs along x as inverse(g) says (float32 steps of 2^-6:
    the map is linear, so differences are exact but for roundings of 2^-24 of the
    sums of 2 * 32 products of normal numbers, below 64 * 16 each)."""
    x, g, table = normal(torch, 9, (3, 2, 32), "float32"), normal(torch, 10, (3, 2, 32), "float32"), table_of(torch, 11, 3, 16)
    for interleaved in (False, True):
        grad = torch.empty_like(g)
        hip.rotary(g, table, grad, interleaved=interleaved, inverse=True)
        for at in [(0, 0, 0), (1, 1, 17), (2, 0, 31), (2, 1, 8)]:
            up, down, e = x.clone(), x.clone(), 2.0 ** -6
            up[at] += e
            down[at] -= e
            outs = []
            for y in (up, down):
                o = torch.empty_like(y)
                hip.rotary(y, table, o, interleaved=interleaved)
                outs.append(float((o.double() * g.double()).sum()))
            assert abs((outs[0] - outs[1]) / (2 * e) - float(grad[at])) <= 192 * 16 * 2.0 ** -24 / e / 16


def test_rotation_keeps_relative_positions(hip, torch):
    """Scores of rotated queries and keys go by the distance of their positions alone."""
    from munet_amd.backend import rotary_frequencies
    freq = torch.from_numpy(rotary_frequencies(64, 10000.0)[0]).cuda()
    q, k = normal(torch, 12, (1, 1, 64), "float32").expand(6, 1, 64).contiguous(), normal(torch, 13, (1, 1, 64), "float32").expand(6, 1, 64).contiguous()
    first = torch.tensor([0, 1, 100, 5000, 100000, 2000000], dtype=torch.int32, device="cuda")
    tq, tk = torch.empty((6, 32, 2), device="cuda"), torch.empty((6, 32, 2), device="cuda")
    hip.rotary_table(first + 37, freq, tq)
    hip.rotary_table(first, freq, tk)
    hip.rotary(q, tq, q)
    hip.rotary(k, tk, k)
    s = (q.double() * k.double()).sum((1, 2))
    size = float((q.double().abs() * k.double().abs()).sum((1, 2)).max()) * 2  # (a rotation moves it by at most 2)
    # each value is off by 2 roundings and its table's two, of 2^-24
    assert float((s - s[0]).abs().max()) <= 2 * 2 * 4 * 2.0 ** -24 * size


# ---- rotated appends -------------------------------------------------------------------

def pool(torch, seed, n_pages, heads, P, hd):
    g = torch.Generator().manual_seed(seed)
    b = lambda s: torch.randint(0, 120, s, generator=g, dtype=torch.uint8).cuda()  # noqa: E731
    sc = lambda: torch.exp2(torch.randint(-9, -2, (n_pages, heads), generator=g).float()).cuda()  # noqa: E731
    return [b((n_pages, heads, P, hd)), b((n_pages, heads, hd, P)), sc(), sc()]


def slots_of(torch, seed, P, n_pages, runs):
    """Runs of (first place, tokens) in pages of their own, some tokens without a slot."""
    pages = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    slots = []
    for first, n in runs:
        g = None
        for t in range(first, first + n):
            if g is None or t % P == 0:
                g = pages.pop()
            slots.append(g * P + t % P)
        slots.append(-1)
    return torch.tensor(slots, dtype=torch.int32, device="cuda")


RUNS = [(0, 1), (5, 1), (3, 70), (0, 16), (15, 2), (0, 200), (9, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("P,kv,heads,hd,rot", [(16, 2, 4, 64, 64), (64, 3, 3, 64, 24), (256, 1, 8, 128, 128), (32, 2, 10, 80, 40), (64, 1, 1, 256, 6),
                                               (128, 2, 2, 256, 256), (16, 1, 5, 16, 16), (16, 2, 4, 128, 120), (32, 2, 3, 128, 100)])
def test_append(hip, torch, dtype, interleaved, P, kv, heads, hd, rot):
    """The cache holds what kv_store_paged makes of the rotated keys in float32, bit for
    bit; queries are rotary()'s; rows without a slot are left alone."""
    n_pages = 60
    slots = slots_of(torch, hd + P, P, n_pages, RUNS)
    n = len(slots)
    rows = normal(torch, P + hd, (n, heads + 2 * kv, hd), dtype)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    table = table_of(torch, hd, n, rot // 2)
    got, want = pool(torch, 1, n_pages, kv, P, hd), pool(torch, 1, n_pages, kv, P, hd)
    q_out = torch.full((n, heads, hd), 3.0, dtype=rows.dtype, device="cuda")
    before = rows.clone()
    hip.kv_store_rotary_paged(k, v, table, slots, *got, q=q, q_out=q_out, interleaved=interleaved)
    assert torch.equal(rows, before)
    turned = torch.empty((n, kv, hd), device="cuda")
    hip.rotary(k.float().contiguous(), table, turned, interleaved=interleaved)
    hip.kv_store_paged(turned, v.float().contiguous(), slots, *want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    q_want = torch.empty_like(q_out)
    hip.rotary(q, table, q_want, interleaved=interleaved)
    q_want[slots < 0] = 3.0
    assert torch.equal(q_out, q_want)
    # without queries, and queries in place
    again = pool(torch, 1, n_pages, kv, P, hd)
    hip.kv_store_rotary_paged(k, v, table, slots, *again, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(again, got))
    again = pool(torch, 1, n_pages, kv, P, hd)
    hip.kv_store_rotary_paged(k, v, table, slots, *again, q=q, q_out=q, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(again, got))
    q_want[slots < 0] = before[:, :heads][slots < 0]
    assert torch.equal(q, q_want) and torch.equal(rows[:, heads:], before[:, heads:])
    hip.check_device_errors()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("P,kv,heads,hd,rot", [(16, 12, 12, 64, 24), (16, 8, 3, 128, 128), (32, 8, 9, 128, 64), (64, 8, 32, 128, 128), (64, 10, 4, 80, 42),
                                               (128, 8, 5, 128, 128), (256, 8, 2, 128, 20), (256, 6, 1, 256, 256), (64, 8, 6, 128, 120),
                                               (32, 8, 7, 128, 100)])
def test_append_prompts(hip, torch, dtype, interleaved, P, kv, heads, hd, rot):
    """Several tokens to a workgroup, workgroups of every size: prompts behind prefixes, some
    tokens without a slot, against the same keys in float32, bit for bit."""
    runs = [(0, 700), (P - 3, 450), (5, 1), (P // 2, 300), (0, P), (1, 2 * P - 1), (0, 333)]
    n_pages = sum(-(-(f + n) // P) for f, n in runs) + 5
    slots = slots_of(torch, hd + P, P, n_pages, runs)
    n = len(slots)
    rows, table = normal(torch, P + hd, (n, heads + 2 * kv, hd), dtype), table_of(torch, hd, n, rot // 2)
    # (sizes that grow along the prompts, so that pages' scales grow behind their prefixes)
    rows *= torch.linspace(0.1, 8.0, n, device="cuda")[:, None, None].to(rows.dtype)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    got, want = pool(torch, 1, n_pages, kv, P, hd), pool(torch, 1, n_pages, kv, P, hd)
    q_out = torch.full((n, heads, hd), 3.0, dtype=rows.dtype, device="cuda")
    hip.kv_store_rotary_paged(k, v, table, slots, *got, q=q, q_out=q_out, interleaved=interleaved)
    turned = torch.empty((n, kv, hd), device="cuda")
    hip.rotary(k.float().contiguous(), table, turned, interleaved=interleaved)
    hip.kv_store_paged(turned, v.float().contiguous(), slots, *want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    q_want = torch.empty_like(q_out)
    hip.rotary(q, table, q_want, interleaved=interleaved)
    q_want[slots < 0] = 3.0
    assert torch.equal(q_out, q_want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_single_tokens_beside_runs(hip, torch, dtype):
    """Batches small enough for a workgroup a token: single tokens at every place of a page, runs
    of two and three, the last token of the call; the same bits as one call a token or run."""
    P, kv, hd, n_pages = 16, 2, 48, 40
    runs = [(i, 1) for i in range(16)] + [(3, 2), (14, 3), (0, 3), (15, 1), (0, 1), (7, 1)]
    slots = slots_of(torch, 5, P, n_pages, runs)[:-1]
    n = len(slots)
    rows = normal(torch, 6, (n, 2, kv, hd), dtype) * 300
    got, want = pool(torch, 7, n_pages, kv, P, hd), pool(torch, 7, n_pages, kv, P, hd)
    hip.kv_store_paged(rows[:, 0], rows[:, 1], slots, *got)
    at = 0
    for _, m in runs:
        hip.kv_store_paged(rows[at:at + m, 0], rows[at:at + m, 1], slots[at:at + m], *want)
        at += m + 1
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # against many tokens to a workgroup: the same rows among enough others
    many = 5000
    filler = torch.full((many,), -1, dtype=torch.int32, device="cuda")
    big, others = torch.cat([slots, filler]), pool(torch, 7, n_pages, kv, P, hd)
    wide = torch.cat([rows, torch.zeros((many, 2, kv, hd), dtype=rows.dtype, device="cuda")])
    hip.kv_store_paged(wide[:, 0], wide[:, 1], big, *others)
    for a, b in zip(got, others):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_against_the_formula(hip, torch, dtype):
    """Keys within half a step of e4m3 (2^-4 of the value, 2^-10 of the scale where it has
    no smaller step) of the rotation in 64 bits, in the least scale that holds them."""
    P, kv, hd = 32, 2, 64
    slots = torch.arange(64, 64 + 90, dtype=torch.int32, device="cuda")
    rows, table = normal(torch, 20, (90, 2 * kv, hd), dtype), table_of(torch, 21, 90, 32)
    kc, vc, ks, vs = pool(torch, 22, 8, kv, P, hd)
    hip.kv_store_rotary_paged(rows[:, :kv], rows[:, kv:], table, slots, kc, vc, ks, vs)
    y, err = rotation(rows[:, :kv], table, False)
    val = e4m3_values(torch)
    for g, a, b in ((2, 0, 32), (3, 32, 64), (4, 64, 90)):
        for h in range(kv):
            scale = float(ks[g, h])
            top = np.abs(y[a:b, h]).max()
            assert scale * 448 >= top * (1 - 2.0 ** -22) and scale * 224 < top * (1 + 2.0 ** -22) and np.log2(scale) % 1 == 0
            held = val[kc[g, h, :b - a].cpu().long()].numpy() * scale
            assert (np.abs(held - y[a:b, h]) <= 2.0 ** -4 * np.abs(y[a:b, h]) + 2.0 ** -10 * scale + 2 * err[a:b, h]).all()


def test_append_refuses_slots_outside_the_pool(hip, torch):
    """They raise the error flag, and their rows of q_out stay."""
    from munet_amd._lib import HipError
    rows, table = normal(torch, 23, (4, 3, 32), "bfloat16"), table_of(torch, 24, 4, 16)
    got = pool(torch, 25, 3, 1, 16, 32)
    before = [t.clone() for t in got]
    q_out = torch.full((4, 1, 32), 3.0, dtype=rows.dtype, device="cuda")
    hip.kv_store_rotary_paged(rows[:, 1:2], rows[:, 2:], table, torch.tensor([-7, 48, 2 ** 31 - 1, 33], dtype=torch.int32, device="cuda"),
                              *got, q=rows[:, :1], q_out=q_out)
    with pytest.raises(HipError, match="out of range"):
        hip.check_device_errors()
    assert (q_out[:3] == 3.0).all() and not (q_out[3] == 3.0).all()
    for a, b in zip(got, before):
        assert torch.equal(a[:2], b[:2])
    hip.check_device_errors()


def test_append_takes_nan(hip, torch):
    """A NaN key marks its pair; the page's scale goes by the others."""
    rows, table = normal(torch, 26, (16, 2, 32), "float16"), table_of(torch, 27, 16, 16)
    rows[4, 0, 5] = float("nan")
    rows[9, 0, 20] = float("inf")
    kc, vc, ks, vs = pool(torch, 28, 2, 1, 16, 32)
    hip.kv_store_rotary_paged(rows[:, :1], rows[:, 1:], table, torch.arange(16, dtype=torch.int32, device="cuda"), kc, vc, ks, vs)
    marks = (kc[0, 0] & 0x7f) == 0x7f
    want = torch.zeros_like(marks)
    want[4, [5, 21]] = want[9, [4, 20]] = True
    assert torch.equal(marks, want)
    y, _ = rotation(rows[:, :1], table, False)
    top = np.abs(y[np.isfinite(y)]).max()
    assert float(ks[0, 0]) * 448 >= top * (1 - 2.0 ** -22) and float(ks[0, 0]) * 224 < top * (1 + 2.0 ** -22)


def test_refusals_of_tensors(hip, torch):
    x, table = normal(torch, 30, (4, 2, 32), "float16"), table_of(torch, 31, 4, 16)
    slots, p = torch.zeros(4, dtype=torch.int32, device="cuda"), pool(torch, 32, 2, 2, 16, 32)
    for call in (lambda: hip.rotary(x, table[:3], x), lambda: hip.rotary(x, table.double(), x), lambda: hip.rotary(x, table, x.float()),
                 lambda: hip.rotary(x.transpose(1, 2), table, x), lambda: hip.rotary(x, table.cpu(), x), lambda: hip.rotary(x[0], table, x),
                 lambda: hip.rotary(x.long(), table, x),
                 lambda: hip.rotary_table(slots.long(), table[:, 0, 0].double(), table),
                 lambda: hip.rotary_table(slots, table[0, :, 0], table),
                 lambda: hip.rotary_table(slots, table[0, :, 0].double(), table[:, :8]),
                 lambda: hip.kv_store_rotary_paged(x, x, table, slots, *p, q=x),
                 lambda: hip.kv_store_rotary_paged(x, x, table, slots[:3], *p),
                 lambda: hip.kv_store_rotary_paged(x, x, table, slots, *p, q=x.float(), q_out=x.float())):
        with pytest.raises(ValueError):
            call()


# ---- graphs and streams ------------------------------------------------------------------

def test_captured_step_with_a_padded_batch(hip, torch):
    """Tables, rotation and appends in one graph, replayed with other tokens, fewer of
    them too, beside eager work on a stream of its own."""
    from munet_amd.backend import rotary_frequencies
    n, kv, heads, hd, P = 48, 2, 4, 64, 16
    freq = torch.from_numpy(rotary_frequencies(hd)[0]).cuda()
    rows = torch.empty((n, heads + 2 * kv, hd), dtype=torch.bfloat16, device="cuda")
    pos, slots = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.full((n,), -1, dtype=torch.int32, device="cuda")
    table, q_out, out = torch.empty((n, hd // 2, 2), device="cuda"), torch.zeros((n, heads, hd), dtype=rows.dtype, device="cuda"), torch.zeros_like(rows)
    cache = pool(torch, 40, 12, kv, P, hd)

    def step(table, cache, q_out, out):
        hip.rotary_table(pos, freq, table)
        hip.rotary(rows, table, out)
        hip.kv_store_rotary_paged(rows[:, heads:heads + kv], rows[:, heads + kv:], table, slots, *cache, q=rows[:, :heads], q_out=q_out)

    side = torch.cuda.Stream()
    rows.normal_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(table, cache, q_out, out)
    mine = [t.clone() for t in cache]
    for turn, live in enumerate([48, 5, 48, 1, 30]):
        rows.copy_(normal(torch, 50 + turn, rows.shape, "bfloat16"))
        pos.copy_(torch.arange(n, dtype=torch.int32) * 31 + turn)
        s = torch.full((n,), -1, dtype=torch.int32)
        s[:live] = torch.arange(live, dtype=torch.int32) + 16 * (turn % 3)
        slots.copy_(s)
        q_out.fill_(turn)
        q_mine = q_out.clone()
        graph.replay()
        torch.cuda.synchronize()
        t2, o2 = torch.empty_like(table), torch.empty_like(out)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            step(t2, mine, q_mine, o2)
        torch.cuda.synchronize()
        assert torch.equal(table, t2) and torch.equal(out, o2) and torch.equal(q_out, q_mine)
        assert all(torch.equal(a, b) for a, b in zip(cache, mine))
        assert (q_out[live:] == turn).all()
    hip.check_device_errors()


def test_append_in_a_pool_past_4_gib(hip, torch):
    """Slots whose bytes lie past 2^32."""
    P, kv, hd = 64, 8, 128
    n_pages = (2 ** 32 // (P * kv * hd)) + 40
    kc = torch.empty((n_pages, kv, P, hd), dtype=torch.uint8, device="cuda")
    vc = torch.empty((n_pages, kv, hd, P), dtype=torch.uint8, device="cuda")
    ks, vs = torch.ones((n_pages, kv), device="cuda"), torch.ones((n_pages, kv), device="cuda")
    last = (n_pages - 2) * P
    slots = torch.arange(last, last + 100, dtype=torch.int32, device="cuda")
    rows, table = normal(torch, 60, (100, 2 * kv, hd), "bfloat16"), table_of(torch, 61, 100, 64)
    small = pool(torch, 62, 2, kv, P, hd)
    hip.kv_store_rotary_paged(rows[:, :kv], rows[:, kv:], table, slots, kc, vc, ks, vs)
    hip.kv_store_rotary_paged(rows[:, :kv], rows[:, kv:], table, slots - last, *small)
    assert torch.equal(kc[-2, :], small[0][0]) and torch.equal(kc[-1, :, :36], small[0][1, :, :36])
    assert torch.equal(vc[-2, :], small[1][0]) and torch.equal(vc[-1, :, :, :36], small[1][1, :, :, :36])
    assert torch.equal(ks[-2:], small[2]) and torch.equal(vs[-2:], small[3])
