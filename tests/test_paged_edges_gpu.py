"""Attention over the paged 8-bit KV cache where its forms meet their ends: joins
of odd cuts, values that are not numbers, masks that differ from wave to wave, pages
nobody wrote.  Against the formula in 64 bits, with the tolerance of
test_paged_gpu.py.  And what the error flag tells."""
import math

import pytest

from test_paged_gpu import DTYPES, E4M3_NAN, Cache, assert_within, attend_reference, check, queries, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd,keys", [(128, 2400), (128, 3000), (80, 2400), (80, 8100), (176, 1500)])
def test_joins_that_leave_threads_over(torch, hip, dtype, hd, keys):  # noqa: F811
    """Head sizes and shares whose product does not divide the joining workgroup."""
    check(torch, hip, Cache(torch, 1, hd, 64, [keys, 70], [1, 1], seed=hd), 2, dtype, what="join")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,P,n,new,window", [(1, 16, 256, 256, 0), (1, 64, 300, 200, 0), (4, 32, 230, 200, 0), (2, 64, 400, 300, 150),
                                                  (4, 128, 261, 261, 90), (1, 16, 333, 290, 200)])
def test_nan_values_in_long_prompts(torch, hip, dtype, heads, P, n, new, window):  # noqa: F811
    """A NaN value reaches every row that sees it, whichever wave's rows the mask ends in."""
    c = Cache(torch, 1, 64, P, [n, 40], [new, 1], seed=P + n, window=window)
    for d, t in ((5, 3), (17, 40), (33, 120), (63, 200), (5, n - 1)):
        c.vc[c.tables[0][t // P], 0, d, t % P] = E4M3_NAN
    out = check(torch, hip, c, heads, dtype, what="NaN values, prompts")
    assert bool(torch.isnan(out).any()) and not bool(torch.isnan(out[:, :, 6]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,P", [(128, 16), (128, 32), (64, 16), (256, 16)])
def test_nan_values_beside_pages_outside_the_pool(torch, hip, dtype, hd, P):  # noqa: F811
    """Marks of an earlier block do not reach rows that see only a later one, part of whose pages is missing."""
    from munet_amd._lib import HipError
    c = Cache(torch, 1, hd, P, [640], [128], seed=hd, window=400)
    c.vc[c.tables[0][144 // P], 0, 5, 144 % P] = E4M3_NAN
    c.vc[c.tables[0][290 // P], 0, 9, 290 % P] = E4M3_NAN
    c.tables[0][256 // P] = -1
    c.sync(torch)
    hip.check_device_errors()
    try:
        check(torch, hip, c, 1, dtype, what="NaN values beside holes")
    finally:
        with pytest.raises(HipError, match="paged KV cache"):
            hip.check_device_errors()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,new,window,causal", [([1, 70, 300, 0], [1, 1, 1, 1], 0, True), ([70, 200, 33], [70, 60, 33], 0, True),
                                                    ([70, 200, 33], [70, 60, 33], 50, True), ([70, 200, 33], [70, 60, 33], 0, False)])
def test_negative_scale(torch, hip, dtype, lens, new, window, causal):  # noqa: F811
    for scale in (-0.125, -2.0):
        check(torch, hip, Cache(torch, 2, 64, 16, lens, new, seed=3, window=window, causal=causal), 4, dtype, what=f"scale {scale}", scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("junk", [math.nan, math.inf, -1.0, 0.0])
@pytest.mark.parametrize("new,P", [(1, 16), (40, 16), (40, 64)])
def test_scales_of_pages_nobody_sees(torch, hip, dtype, junk, new, P):  # noqa: F811
    """Page 0, which no table names, and pages behind the window may hold anything as scales."""
    from munet_amd._lib import HipError
    c = Cache(torch, 2, 64, P, [300, 90], [new, new], seed=7, window=100)
    c.kc, c.vc = (torch.cat([torch.full_like(x[:1], E4M3_NAN), x]) for x in (c.kc, c.vc))
    c.ks, c.vs = (torch.cat([torch.full_like(x[:1], junk), x]) for x in (c.ks, c.vs))
    c.n_pages += 1
    c.tables = [[p + 1 if p >= 0 else p for p in row] for row in c.tables]
    behind = c.tables[0][:(300 - new - 100 + 1) // P]
    c.ks[behind], c.vs[behind] = junk, junk
    c.tables[0][-1 if P == 16 else 3] = -1
    c.sync(torch)
    check(torch, hip, c, 4, dtype, what="scales nobody sees")
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()


@pytest.mark.parametrize("P,window", [(16, 20), (32, 20), (16, 70), (64, 90)])
@pytest.mark.parametrize("new", [1, 20])
def test_pages_behind_the_window_may_be_gone(torch, hip, P, window, new):  # noqa: F811
    """Entries before the first key that a query sees are no error, and the page of that key is one."""
    from munet_amd._lib import HipError
    c = Cache(torch, 2, 64, P, [200, 127], [new, new], window=window, seed=P)
    first = [max(n - new - window + 1, 0) // P for n in c.lens]
    for row, p in zip(c.tables, first):
        row[:p] = [-1 - i for i in range(p)]
    c.sync(torch)
    hip.check_device_errors()
    check(torch, hip, c, 4, "bfloat16", what="pages behind the window")
    hip.check_device_errors()
    c.tables[0][first[0]] = -1
    c.sync(torch)
    check(torch, hip, c, 4, "bfloat16", what="the window's first page")
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()


def _small_pool(torch):
    kc, vc = (torch.zeros((3, 1, 16, 16), dtype=torch.uint8, device="cuda") for _ in range(2))
    return kc, vc, torch.ones((3, 1), device="cuda"), torch.ones((3, 1), device="cuda")


@pytest.mark.parametrize("slot", [-2, -2 ** 31, 48])
def test_slots_outside_the_pool_raise(torch, hip, slot):  # noqa: F811
    """Any but -1, which is skipped in silence."""
    from munet_amd._lib import HipError
    x, pool = torch.ones((3, 1, 16), device="cuda"), _small_pool(torch)
    slots = lambda *s: torch.tensor(s, dtype=torch.int32, device="cuda")  # noqa: E731
    hip.kv_store_paged(x, x, slots(-1, 5, -1), *pool)
    hip.check_device_errors()
    hip.kv_store_paged(x, x, slots(-1, slot, 6), *pool)
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()
    assert pool[0][0].any(-1)[0].nonzero().flatten().tolist() == [5, 6] and not bool(pool[0][1:].any())


def test_engine_runs_go_on(torch, hip):  # noqa: F811
    """An error of the paged calls is not the engine's, and neither takes the other's away."""
    from munet_amd import models
    from munet_amd._lib import HipError
    from munet_amd.engine import Engine
    cfg = models.decoder_config(vocab=100, ctx=16, d_model=64, num_heads=2, num_layers=1, ffn=128)
    eng = Engine(0).load(cfg, models.init_params(cfg, "gpt", scope="p")).compile((1, 16))
    ids = models.make_input(cfg, (1, 16), "gpt", scope="p_in")
    before, x = eng.run(ids), torch.ones((1, 1, 16), device="cuda")
    hip.kv_store_paged(x, x, torch.tensor([48], dtype=torch.int32, device="cuda"), *_small_pool(torch))
    assert (eng.run(ids) == before).all()
    bad = ids.copy()
    bad[0, 3] = 100
    with pytest.raises(HipError, match="Embedding index out of range"):
        eng.run(bad)
    with pytest.raises(HipError, match="paged KV cache"):
        hip.check_device_errors()
    hip.check_device_errors()
    assert (eng.run(ids) == before).all()


def test_all_errors_are_told(torch, hip):  # noqa: F811
    """A plan that runs out of pages, the attention over its table and a bad token id, checked once."""
    from munet_amd._lib import HipError
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    c = Cache(torch, 1, 64, 16, [20], [1], junk=False)
    tables, total, cu, slots, used = i32(0, -1, -1)[None], i32(0), i32(0, 0), i32(*[0] * 20), i32(0)
    hip.check_device_errors()
    hip.page_plan(i32(10), i32(20), i32(), tables, total, cu, slots, None, used, 16, c.n_pages)
    q = queries(torch, 20, 1, 64, "bfloat16")
    hip.attention_paged(q, c.kc, c.vc, c.ks, c.vs, tables, total, cu, torch.empty_like(q), 20, 30)
    w = torch.zeros((10, 8), device="cuda")
    hip.embedding(i32(1, 10, 3), w, torch.zeros((3, 8), device="cuda"), 3, 10, 8)
    with pytest.raises(HipError) as e:
        hip.check_device_errors()
    for what in ("Embedding index", "page_plan", "paged KV cache"):
        assert what in str(e.value)
    hip.check_device_errors()


def test_bounds_past_a_launch(torch, hip):  # noqa: F811
    """Bounds that ask for more workgroups than a launch has: fewer, which walk."""
    B, heads, kv, n_rows = 256, 64, 8, 65600
    lens, new = [300] + [1 + 3 * i for i in range(B - 1)], [300] + [1] * (B - 1)
    c = Cache(torch, kv, 16, 16, lens, new, seed=12)
    q = queries(torch, n_rows, heads, 16, "bfloat16")
    out, rows = torch.full_like(q, 7.0), c.cu[-1]
    ref, tol = attend_reference(torch, c, q[:rows], out[:rows])
    c.attend(hip, q, out, max_q=n_rows, max_len=n_rows)
    assert_within(torch, out[:rows], ref, tol, "many workgroups")
    assert bool((out[rows:] == 7.0).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("low,high", [(-100, 30), (-100, 90), (-100, 28)])
def test_zero_pages_beside_large_values(torch, hip, dtype, new, P, low, high):  # noqa: F811
    """Pages of zeros (scale 2^-100) beside large values: their weights stay in the sum."""
    c = Cache(torch, 2, 64, P, [200, 90, 64], [new, new, 1], seed=4, spread=1.0)
    c.vs[:] = 2.0 ** high
    for b, p in ((0, 0), (0, 2), (1, 1), (2, 0)):
        g = c.tables[b][p]
        c.vs[g] = 2.0 ** low
        c.vc[g] = torch.where(c.vc[g] == E4M3_NAN, E4M3_NAN, 0).to(torch.uint8)
    check(torch, hip, c, 4, dtype, what="zero pages")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("lens,new", [([200, 90, 64], [1, 1, 1]), ([200, 90, 64], [40, 40, 1]), ([3000, 700], [1, 1]), ([900, 700], [40, 1])])
def test_values_near_the_largest(torch, hip, dtype, lens, new):  # noqa: F811
    """Outputs that a float holds, and whose products with the softmax's sum it does not, in one share and joined ones."""
    for P in (16, 64):
        c = Cache(torch, 1, 64, P, lens, new, seed=4, spread=1.0)
        c.vs[:] = 2.0 ** 118
        c.vs[c.tables[0][1]] = 2.0 ** -12
        check(torch, hip, c, 2, dtype, what="large values")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("apart", [20, 40, 100])
def test_large_values_of_no_weight(torch, hip, dtype, new, P, apart):  # noqa: F811
    """Pages of values 2^apart larger, whose scores lie 56 (168) below the others', leave the others' precision alone."""
    low = -9 if dtype == "float16" else -30  # (an fp16 output stays above its type's least step)
    c = Cache(torch, 2, 64, P, [300, 150], [new, new], seed=5, spread=1.0)
    c.ks[:], c.vs[:] = 2.0 ** -6, 2.0 ** low
    c.kc[..., 0] = torch.where(c.kc[..., 0] == E4M3_NAN, E4M3_NAN, 0).to(torch.uint8)
    for b, p in ((0, 0), (0, 3), (1, 1)):
        g = c.tables[b][p]
        c.vs[g] = 2.0 ** (apart + low)
        c.kc[g, :, :, 0] = torch.where(c.kc[g, :, :, 0] == E4M3_NAN, E4M3_NAN, 0xFE).to(torch.uint8)  # -448
    q = queries(torch, c.cu[-1], 4, 64, dtype)
    q[:, :, 0] = 8.0 if apart < 100 else 24.0
    out = torch.full_like(q, 7.0)
    ref, tol = attend_reference(torch, c, q, out, 1.0)
    c.attend(hip, q, out, scale=1.0)
    assert_within(torch, out, ref, tol, "large values of no weight")
