"""Rows in 8-bit integers and the products of them on the GPU.

Rounding to whole numbers is exact: 127 x and its quotient by the row's largest
magnitude, in 64 bits, tell every tie.

Tolerance of linear_i8, with v = sx sw S (S the exact sum): S as float32 and two
products, 2^-24 each, and where v is below the normal numbers a step of 2^-149;
the bias another 2^-24 of their sum.  GELU v sigmoid(1.702 v): the slope is at
most 1.2; the argument's product with 1.702 and with log2 e and the constants
themselves are off by 2^-24 each, which the exponential multiplies by the
argument, and exponential, sum and reciprocal by 2 units of the last place each:
(4 |1.702 v| + 16) 2^-24 of the result, and 2^-118 where the exponential leaves the
range.  The residual adds 2^-24 of the sum, the output half a step of its type."""
import numpy as np
import pytest

from test_paged_gpu import DTYPES, HALF_STEP
from test_rotary_gpu import LEAST, normal, pool, rotation, check as check_rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch(hip):
    import torch as t
    from munet_amd._lib import HipError
    try:  # (errors that tests of other files left set)
        hip.check_device_errors()
    except HipError:
        pass
    return t


# ---- rows ----------------------------------------------------------------------------

def rows_reference(x):
    """(whole numbers, scales) of float64 rows of values that are floats."""
    a = np.maximum(np.abs(x).max(1), 127 * 2.0 ** -126)
    return np.rint(127 * x / a[:, None]), (a / 127).astype(np.float32)


def check_rows(hip, torch, x):
    n, c = x.shape
    q, s = torch.full((n + 1, c), 99, dtype=torch.int8, device="cuda"), torch.full((n + 1,), 7.0, device="cuda")
    hip.quantize_rows(x, q[:n], s[:n])
    want, scale = rows_reference(x.double().cpu().numpy())
    got = q[:n].cpu().numpy()
    assert (got == want).all(), (int((got != want).sum()), np.argwhere(got != want)[:4])
    assert (s[:n].cpu().numpy() == scale).all()
    assert (q[n] == 99).all() and s[n] == 7.0
    for dtype in DTYPES:
        out = torch.full((n + 1, c), 5.0, dtype=getattr(torch, dtype), device="cuda")
        hip.dequantize_rows(q[:n], s[:n], out[:n])
        v = want * scale.astype(np.float64)[:, None]
        off = np.abs(out[:n].double().cpu().numpy() - v)
        fits = np.abs(v) < (65000 if dtype == "float16" else 3e38)
        # the product in float32, then the output type
        assert (off <= 2.0 ** -24 * np.abs(v) + HALF_STEP[dtype] * np.abs(v) * (1 + 2.0 ** -20) + LEAST[dtype] + 2.0 ** -149)[fits].all()
        assert (out[n] == 5.0).all()
    return q[:n], s[:n]


ROWS = [(1, 1), (1, 7), (3, 8), (5, 63), (2, 64), (64, 768), (7, 1001), (9, 2048), (3, 2049), (2, 4096), (5, 8192), (3, 8200), (2, 16384), (2, 32768),
        (1, 32775), (2, 70001), (1000, 33), (4099, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", ROWS)
def test_rows(hip, torch, dtype, n, c):
    check_rows(hip, torch, normal(torch, n + c, (n, c), dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [1.0, 127.0, 254.0, 0.49609375])
def test_ties(hip, torch, dtype, top):
    """Rows whose quotients lie on halves (a largest value of 127 2^k), and next to them."""
    k = torch.arange(-254, 255, dtype=torch.float64)
    x = k / 254 * top
    x = torch.stack([x, torch.nextafter(x.float(), torch.tensor(9e9)).double().clamp(-top, top),
                     torch.nextafter(x.float(), torch.tensor(-9e9)).double().clamp(-top, top)])
    x = x.to(getattr(torch, dtype)).cuda()
    x[:, 0], x[:, -1] = -top, top
    check_rows(hip, torch, x)


def test_rows_near_halves_in_float32(hip, torch):
    """The floats next to every half of rows of odd largest values."""
    tops = torch.tensor([1.0000001, 1.3333334, 2.7182817, 1e-30, 3.4e38, 1.5e-36], dtype=torch.float64)
    x = []
    for a in tops.float().tolist():
        h = ((torch.arange(-127, 127) + 0.5) * (a / 127)).float()
        x.append(torch.cat([h, torch.nextafter(h, torch.tensor(float("inf"))), torch.nextafter(h, torch.tensor(float("-inf")))]).clamp(-a, a))
        x[-1][0] = a
    check_rows(hip, torch, torch.stack(x).cuda())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_extremes(hip, torch, dtype):
    """Zeros, the smallest values, the largest."""
    f = torch.finfo(getattr(torch, dtype))
    x = torch.zeros((5, 70))
    x[1, 3] = -f.tiny
    x[2] = torch.arange(70) * f.smallest_normal / 64
    x[3] = torch.linspace(-1, 1, 70) * f.max
    x[4, 69] = 1e-3
    check_rows(hip, torch, x.to(getattr(torch, dtype)).cuda())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [5, 64, 9000])
def test_rows_that_are_not_finite(hip, torch, dtype, c):
    x = normal(torch, 3, (6, c), dtype)
    x[1, c - 1], x[2, 0], x[4, c // 2] = float("nan"), float("inf"), float("-inf")
    q, s = torch.full((6, c), 99, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    hip.quantize_rows(x, q, s)
    assert s.isnan().tolist() == [False, True, True, False, True, False]
    assert not q[[1, 2, 4]].any() and q[[0, 3, 5]].any()
    out = torch.empty_like(x)
    hip.dequantize_rows(q, s, out)
    assert out[[1, 2, 4]].isnan().all() and not out[[0, 3, 5]].isnan().any()
    y, w = torch.empty((6, 3), device="cuda"), torch.ones((3, c), dtype=torch.int8, device="cuda")
    for act in (0, 1, 2):
        hip.linear_i8(q, s, w, torch.ones(3, device="cuda"), y, act=act)
        assert y[[1, 2, 4]].isnan().all() and not y[[0, 3, 5]].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,ld,first", [(64, 80, 16), (61, 77, 3), (1000, 1008, 0), (2050, 2051, 1)])
def test_rows_of_views(hip, torch, dtype, c, ld, first):
    """Columns of wider rows, at any alignment; what lies beside them stays."""
    wide, n = normal(torch, 4, (13, ld), dtype), 13
    q = torch.full((n, ld + 5), 99, dtype=torch.int8, device="cuda")
    s = torch.empty(n, device="cuda")
    hip.quantize_rows(wide[:, first:first + c], q[:, 5:5 + c], s)
    want, scale = rows_reference(wide[:, first:first + c].double().cpu().numpy())
    assert (q[:, 5:5 + c].cpu().numpy() == want).all() and (s.cpu().numpy() == scale).all()
    assert (q[:, :5] == 99).all() and (q[:, 5 + c:] == 99).all()
    out = torch.full((n, ld), 5.0, dtype=wide.dtype, device="cuda")
    hip.dequantize_rows(q[:, 5:5 + c], s, out[:, first:first + c])
    packed = torch.empty((n, c), dtype=wide.dtype, device="cuda")
    hip.dequantize_rows(q[:, 5:5 + c].contiguous(), s, packed)
    assert torch.equal(out[:, first:first + c], packed)
    assert (out[:, :first] == 5.0).all() and (out[:, first + c:] == 5.0).all()


# ---- products -------------------------------------------------------------------------

def linear_reference(x, sx, w, sw, bias, act, resid):
    """(value, what roundings in float32 may add) in 64 bits."""
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    u = 2.0 ** -24
    # (whole numbers below 2^53 are exact in float64)
    v = (f(x) @ f(w).T) * f(sx)[:, None] * f(sw)
    err = 3 * u * np.abs(v) * (1 + 2.0 ** -20) + 2.0 ** -149
    if bias is not None:
        v = v + f(bias)
        err += u * (np.abs(v) + err)
    if act == 1:
        v = np.maximum(v, 0)
    elif act == 2:
        with np.errstate(over="ignore"):
            g = v / (1 + np.exp(-1.702 * v))
        err = 1.2 * err + (4 * np.abs(1.702 * v) + 16) * u * np.abs(g) + 2.0 ** -118
        v = g
    if resid is not None:
        v = v + f(resid)
        err += u * (np.abs(v) + err)
    return v, err


def check_linear(hip, torch, x, sx, w, sw, dtype, bias=None, act=0, resid=None, out=None):
    M, N = x.shape[0], w.shape[0]
    if out is None:
        out = torch.full((M + 1, N), 5.0, dtype=getattr(torch, dtype), device="cuda")
    v, err = linear_reference(x, sx, w, sw, bias, act, resid)
    hip.linear_i8(x, sx, w, sw, out[:M], bias=bias, act=act, resid=resid)
    got = out[:M].double().cpu().numpy()
    bad = ~(np.abs(got - v) <= err + HALF_STEP[dtype] * (np.abs(v) + err) + LEAST[dtype])
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], v[bad][:4])
    if out.shape[0] > M:
        assert (out[M] == 5.0).all()
    return out[:M]


def operands(torch, seed, M, N, K):
    g = torch.Generator().manual_seed(seed)
    i = lambda r: torch.randint(-128, 128, (r, K), generator=g, dtype=torch.int8).cuda()  # noqa: E731
    s = lambda r: (torch.rand(r, generator=g) * 0.02 + 1e-4).cuda()  # noqa: E731
    return i(M), s(M), i(N), s(N)


PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 768, 768), (2, 100, 64), (3, 33, 1001), (4, 257, 4096), (5, 64, 130), (8, 1000, 768), (15, 17, 127), (16, 64, 128),
            (17, 80, 144), (31, 130, 272), (33, 100, 500), (64, 64, 64), (64, 520, 1040), (65, 129, 257), (100, 1, 256), (128, 128, 384),
            (129, 255, 640), (200, 3, 2000), (257, 300, 192), (256, 512, 4096), (500, 700, 96), (1, 5000, 48), (1000, 24, 1024), (513, 1025, 160)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_linear(hip, torch, dtype, M, N, K):
    x, sx, w, sw = operands(torch, M + N + K, M, N, K)
    check_linear(hip, torch, x, sx, w, sw, dtype)
    bias, resid = normal(torch, 1, (N,), dtype), normal(torch, 2, (M, N), dtype)
    check_linear(hip, torch, x, sx, w, sw, dtype, bias=bias, act=(M + N) % 3, resid=resid)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 260, 320), (7, 36, 96), (40, 72, 200), (150, 260, 512)])
@pytest.mark.parametrize("act", [0, 1, 2])
def test_linear_epilogues(hip, torch, dtype, M, N, K, act):
    x, sx, w, sw = operands(torch, K, M, N, K)
    bias, resid = normal(torch, 1, (N,), dtype), normal(torch, 2, (M, N), dtype)
    for b in (None, bias):
        for r in (None, resid):
            got = check_linear(hip, torch, x, sx, w, sw, dtype, bias=b, act=act, resid=r)
    # the residual in place, the same bits
    y = resid.clone()
    hip.linear_i8(x, sx, w, sw, y, bias=bias, act=act, resid=y)
    assert torch.equal(y, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 6, 30, 100, 300])
@pytest.mark.parametrize("K,ldx,ldw,fx,fw", [(100, 112, 128, 0, 0), (128, 144, 160, 16, 32), (77, 90, 83, 3, 5), (1000, 1008, 1024, 0, 16), (64, 65, 71, 1, 7)])
def test_linear_of_views(hip, torch, dtype, M, K, ldx, ldw, fx, fw):
    """Columns of wider rows: what lies beside them in the operands does not count, beside
    the output it stays."""
    N = 90
    x, sx, w, sw = operands(torch, K + M, M, N, ldx)
    w = torch.randint(-128, 128, (N, ldw), generator=torch.Generator().manual_seed(1), dtype=torch.int8).cuda()
    xv, wv = x[:, fx:fx + K], w[:, fw:fw + K]
    for first, ldo in ((4, 104), (3, 97)):
        wide, res = torch.full((M, ldo), 5.0, dtype=getattr(torch, dtype), device="cuda"), normal(torch, 3, (M, ldo + 1), dtype)
        check_linear(hip, torch, xv, sx, wv, sw, dtype, bias=normal(torch, 4, (N + 1,), dtype)[1:], resid=res[:, 2:2 + N], out=wide[:, first:first + N])
        assert (wide[:, :first] == 5.0).all() and (wide[:, first + N:] == 5.0).all()


KERNELS = [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 100, 101]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("M,N,K", [(1, 40, 16), (70, 264, 208), (256, 300, 1040), (200, 257, 128)])
def test_every_kernel(hip, torch, monkeypatch, kernel, dtype, M, N, K):
    """Each kernel and tile on sizes off its own, against the formula; and the bits of the one
    that the sizes choose."""
    x, sx, w, sw = operands(torch, M + K, M, N, K)
    bias, resid = normal(torch, 1, (N,), dtype), normal(torch, 2, (M, N), dtype)
    for act, r in ((0, resid), (1, None), (2, resid)):
        own = torch.empty((M, N), dtype=resid.dtype, device="cuda")
        hip.linear_i8(x, sx, w, sw, own, bias=bias, act=act, resid=r)
        with monkeypatch.context() as m:
            m.setenv("MUNET_HIP_I8_TILE", str(kernel))
            got = check_linear(hip, torch, x, sx, w, sw, dtype, bias=bias, act=act, resid=r)
        assert torch.equal(got, own)


@pytest.mark.parametrize("kernel", [0, 10, 100, 101])
@pytest.mark.parametrize("K,ldx,ldw,fx,fw", [(1, 3, 5, 1, 2), (15, 21, 18, 2, 3), (65, 70, 66, 5, 1), (130, 131, 137, 0, 7), (255, 259, 260, 3, 4), (1027, 1030, 1031, 1, 2)])
def test_kernels_of_unaligned_rows(hip, torch, monkeypatch, kernel, K, ldx, ldw, fx, fw):
    """Rows at every offset from a word, ends inside one."""
    monkeypatch.setenv("MUNET_HIP_I8_TILE", str(kernel))
    x, sx, _, _ = operands(torch, K, 37, 1, ldx)
    w, sw, _, _ = operands(torch, K + 1, 150, 1, ldw)
    check_linear(hip, torch, x[:, fx:fx + K], sx, w[:, fw:fw + K], sw, "float32")


@pytest.mark.parametrize("M", [1, 16, 70])
def test_linear_sums_fill_32_bits(hip, torch, M):
    """The longest rows of the lowest value: sums of 2^31 - 2^14; and of both signs."""
    K, N = 2 ** 17 - 1, 20
    x, w = torch.full((M, K), -128, dtype=torch.int8, device="cuda"), torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    w[1], w[2, ::2] = 127, 127
    one = torch.ones(max(M, N), device="cuda")
    check_linear(hip, torch, x, one[:M], w, one[:N], "float32")


@pytest.mark.parametrize("M", [1, 40])
def test_linear_scales_of_any_size(hip, torch, M):
    """Products of scales outside the floats with results inside; zeros, infinities and NaN."""
    x, _, w, _ = operands(torch, 5, M, 8, 256)
    x[:, 0] = 1
    sx = torch.tensor([2.0 ** (127 - i % 3 * 254 if i % 3 < 2 else -149) for i in range(M)], device="cuda")
    sw = torch.tensor([2.0 ** -149, 2.0 ** -126, 1e-30, 1.0, 2.0 ** 100, 0.0, 3e38, 1e-20], device="cuda")
    v, err = linear_reference(x, sx, w, sw, None, 0, None)
    out = torch.empty((M, 8), device="cuda")
    hip.linear_i8(x, sx, w, sw, out)
    got = out.double().cpu().numpy()
    fits = np.abs(v) < 3.4e38
    assert (np.abs(got - v) <= err + HALF_STEP["float32"] * np.abs(v) + 2.0 ** -149)[fits].all()
    assert np.isinf(got[~fits & (np.abs(v) > 3.41e38)]).all()
    sx[0], sw[3] = float("nan"), float("nan")
    hip.linear_i8(x, sx, w, sw, out)
    assert out[0].isnan().all() and out[:, 3].isnan().all() and not out[1:, [0, 1, 2, 4]].isnan().any()


def test_linear_outputs_past_2_gib(hip, torch):
    """Outputs and weights whose offsets pass 2^31 and 2^32 bytes, against the same rows in small."""
    N, K, M = 40000, 80, 60000
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device="cuda")
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device="cuda")
    sx, sw = torch.rand(M, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    out = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    hip.linear_i8(x, sx, w, sw, out)
    for rows in (slice(0, 70), slice(30000, 30070), slice(M - 70, M)):
        check_linear(hip, torch, x[rows], sx[rows], w, sw, "bfloat16", out=out[rows].clone())
        small = torch.empty((70, N), dtype=torch.bfloat16, device="cuda")
        hip.linear_i8(x[rows], sx[rows], w, sw, small)
        assert torch.equal(out[rows], small)


def test_linear_far_rows(hip, torch):
    """Rows of operands gigabytes apart."""
    buf = torch.empty(5 * 2 ** 30, dtype=torch.int8, device="cuda")
    K, N = 512, 20
    for M in (2, 40):
        far = buf.as_strided((M, K), (5 * 2 ** 30 // M // 16 * 16, 1))
        x, sx, w, sw = operands(torch, M, M, N, K)
        far.copy_(x)
        check_linear(hip, torch, far, sx, w, sw, "float16")
        far = buf.as_strided((N, K), (5 * 2 ** 30 // N // 16 * 16, 1))
        far.copy_(w)
        check_linear(hip, torch, x, sx, far, sw, "float16")


def test_refusals_of_tensors(hip, torch):
    x, sx, w, sw = operands(torch, 9, 4, 6, 32)
    out, f = torch.empty((4, 6), device="cuda"), torch.empty((4, 32), device="cuda")
    for call in (lambda: hip.linear_i8(x, sx[:3], w, sw, out), lambda: hip.linear_i8(x, sx, w[:, :16], sw, out),
                 lambda: hip.linear_i8(x, sx, w, sw, out[:, :5]), lambda: hip.linear_i8(x.float(), sx, w, sw, out),
                 lambda: hip.linear_i8(x, sx.double(), w, sw, out), lambda: hip.linear_i8(x, sx, w, sw, out, bias=sw.half()),
                 lambda: hip.linear_i8(x, sx, w, sw, out, resid=out.half()), lambda: hip.linear_i8(x, sx, w, sw, out.int()),
                 lambda: hip.linear_i8(x.t(), sx, w, sw, out), lambda: hip.linear_i8(x, sx, w.cpu(), sw, out),
                 lambda: hip.linear_i8(x, sx[:1].expand(4), w, sw, out),
                 lambda: hip.quantize_rows(f, x.t(), sx), lambda: hip.quantize_rows(f.int(), x, sx), lambda: hip.quantize_rows(f, x, sx.double()),
                 lambda: hip.quantize_rows(f, x[:, :16], sx), lambda: hip.dequantize_rows(x, sx, f[:3]), lambda: hip.dequantize_rows(f, sx, f),
                 lambda: hip.dequantize_rows(x, sx, x)):
        with pytest.raises(ValueError):
            call()


# ---- a layer --------------------------------------------------------------------------

class Layer:
    """A decoder layer's attention in 8 bits over the paged cache, as a server runs it."""

    def __init__(self, torch, hip, seed, d, heads, kv, hd, n, dtype):
        self.hip, self.n, self.heads, self.kv, self.hd, self.d = hip, n, heads, kv, hd, d
        out = (heads + 2 * kv) * hd
        t = getattr(torch, dtype)
        e = lambda s, ty=t: torch.zeros(s, dtype=ty, device="cuda")  # noqa: E731
        self.weights = []
        for o, i in ((out, d), (d, heads * hd)):
            w, q, s = normal(torch, seed + o, (o, i), dtype) / i ** 0.5, e((o, i), torch.int8), e((o,), torch.float32)
            hip.quantize_rows(w, q, s)
            self.weights.append((q, s))
        self.bias = normal(torch, seed, (out,), dtype)
        self.x8, self.a8, self.s1, self.s2 = e((n, d), torch.int8), e((n, heads * hd), torch.int8), e((n,), torch.float32), e((n,), torch.float32)
        self.rows, self.q, self.att, self.out = e((n, heads + 2 * kv, hd)), e((n, heads, hd)), e((n, heads, hd)), e((n, d))

    def __call__(self, x, table, slots, cache, tables, total, cu, max_q, max_len, ws):
        h, H, KV = self.hip, self.heads, self.kv
        h.quantize_rows(x, self.x8, self.s1)
        h.linear_i8(self.x8, self.s1, *self.weights[0], self.rows.view(self.n, -1), bias=self.bias)
        h.kv_store_rotary_paged(self.rows[:, H:H + KV], self.rows[:, H + KV:], table, slots, *cache, q=self.rows[:, :H], q_out=self.q)
        h.attention_paged(self.q, *cache, tables, total, cu, self.att, max_q, max_len, workspace=ws)
        h.quantize_rows(self.att.view(self.n, -1), self.a8, self.s2)
        h.linear_i8(self.a8, self.s2, *self.weights[1], self.out, resid=x)
        return self.out


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_layer(hip, torch, dtype):
    """Three steps of ragged requests (prompts, then tokens), each stage against its formula on
    what the stage before left; then the last step captured and replayed."""
    from munet_amd.backend import rotary_frequencies
    from test_paged_gpu import e4m3_values
    d, heads, kv, hd, P, B, n_pages = 256, 8, 2, 64, 16, 3, 40
    freq, mag = rotary_frequencies(hd)
    freq = torch.from_numpy(freq).cuda()
    cache = [t.zero_() for t in pool(torch, 70, n_pages, kv, P, hd)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, free = [0, 0, 0], list(range(n_pages))
    tables = torch.full((B, 8), -1, dtype=torch.int32, device="cuda")
    # one step of prompts, two of single tokens
    for step, new in enumerate([[50, 1, 17], [1, 1, 1], [1, 1, 1]]):
        n = sum(new)
        total, cu, slots, pos, used = i32([0] * B), i32([0] * (B + 1)), i32([0] * n), i32([0] * n), i32([0])
        hip.page_plan(i32(lens), i32(new), i32(free), tables, total, cu, slots, pos, used, P, n_pages)
        free, lens = free[int(used):], total.tolist()
        table = torch.empty((n, hd // 2, 2), device="cuda")
        hip.rotary_table(pos, freq, table, magnitude=mag)
        layer, x = Layer(torch, hip, 71, d, heads, kv, hd, n, dtype), normal(torch, 72 + step, (n, d), dtype)
        ws = torch.empty(hip.attention_paged_workspace(layer.q, cache[0], total, max(new), 128), dtype=torch.uint8, device="cuda")
        args = (x, table, slots, cache, tables, total, cu, max(new), 128, ws)
        out = layer(*args).clone()
        hip.check_device_errors()
        # the product of the rounded rows
        v, err = linear_reference(layer.x8, layer.s1, *layer.weights[0], layer.bias, 0, None)
        got = layer.rows.view(n, -1).double().cpu().numpy()
        assert (np.abs(got - v) <= err + HALF_STEP[dtype] * (np.abs(v) + err) + LEAST[dtype]).all()
        check_rotated(layer.q, *rotation(layer.rows[:, :heads], table, False), dtype)
        # the cache's new keys: e4m3 of the rotated ones
        y, e = rotation(layer.rows[:, heads:heads + kv], table, False)
        val, sl = e4m3_values(torch), slots.cpu().long()
        scale = cache[2].cpu().double()[sl // P]
        held = val[cache[0].cpu().long()[sl // P, :, sl % P]] * scale[..., None]
        held, scale = held.numpy(), scale.numpy()[..., None]
        assert (np.abs(held - y) <= 2.0 ** -4 * np.abs(y) + 2.0 ** -10 * scale + 2 * e).all()
        v, err = linear_reference(layer.a8, layer.s2, *layer.weights[1], None, 0, x)
        assert (np.abs(out.double().cpu().numpy() - v) <= err + HALF_STEP[dtype] * (np.abs(v) + err) + LEAST[dtype]).all()
    # the same step again leaves the same cache; captured, it gives the same bits
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        layer(*args)
    for turn in range(4):
        x.copy_(normal(torch, 90 + turn, x.shape, dtype))
        graph.replay()
        torch.cuda.synchronize()
        got, mine = layer.out.clone(), [t.clone() for t in cache]
        assert torch.equal(layer(*args), got)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cache, mine))
