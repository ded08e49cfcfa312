"""Operands of the rotated append that share bytes with the pages and scales it writes: refused
by name, on the CPU; operands right beside them are taken."""
import pytest

from munet_amd import _lib

PAGES, HKV, HD, PAGE, N, HQ = 16, 8, 128, 64, 4, 32
POOL, SCALE, ROW, QROW = PAGES * HKV * PAGE * HD, PAGES * HKV * 4, HKV * HD * 2, HQ * HD * 2
AT = {name: (i + 1) << 32 for i, name in enumerate(["k", "v", "table", "slots", "kc", "vc", "ks", "vs", "q", "q_out"])}


def _store(**kw):
    a = dict(dt=2, k=0, v=0, ldk=HKV * HD, ldv=HKV * HD, table=0, slots=0, kc=0, vc=0, ks=0, vs=0, n=N, Hkv=HKV, hd=HD, half=64, inter=0,
             page=PAGE, n_pages=PAGES, q=0, ldq=HQ * HD, q_out=0, ldqo=HQ * HD, Hq=HQ)
    a.update(AT)
    a.update(kw)
    _lib.call("mh_kv_store_rotary_paged", *a.values(), None)


@pytest.mark.parametrize("pool,size", [("kc", POOL), ("vc", POOL), ("ks", SCALE), ("vs", SCALE)])
@pytest.mark.parametrize("other,bytes_", [("q_out", N * QROW), ("q", N * QROW), ("k", N * ROW), ("v", N * ROW), ("table", N * 64 * 8), ("slots", N * 4)])
def test_operands_over_pages_and_scales(pool, size, other, bytes_):
    assert size % 16 == 0 and bytes_ % 16 == 0
    for at in (AT[pool], AT[pool] + size - 16, AT[pool] + size // 32 * 16, AT[pool] - bytes_ + 16):
        kw = {other: at}
        if other == "q_out":  # queries in place too
            with pytest.raises(_lib.HipError, match="overlap a cache or a scale"):
                _store(q=at, q_out=at)
        with pytest.raises(_lib.HipError, match="overlap a cache or a scale"):
            _store(**kw)
        if other in ("k", "v", "table", "slots"):
            with pytest.raises(_lib.HipError, match="overlap a cache or a scale"):
                _store(**kw, q=None, q_out=None)


def test_pages_and_scales_over_each_other():
    names = {"kc": POOL, "vc": POOL, "ks": SCALE, "vs": SCALE}
    for a, size in names.items():
        for b in names:
            if a != b:
                with pytest.raises(_lib.HipError, match="caches and scales overlap"):
                    _store(**{b: AT[a] + size - 16})


def test_rows_too_far_apart_without_queries():
    for kw in (dict(ldk=1 << 58), dict(ldv=1 << 58)):
        with pytest.raises(_lib.HipError, match="far apart"):
            _store(**kw, q=None, q_out=None)


@pytest.mark.gpu
def test_operands_beside_pages_and_scales(hip):
    """Everything in one buffer, one behind the other: taken, and the same as in buffers of their own."""
    import torch
    pages, kv, P, hd, n, heads = 3, 2, 16, 32, 5, 4
    g = torch.Generator().manual_seed(1)
    rows = torch.randn((n, heads + 2 * kv, hd), generator=g).bfloat16().cuda()
    table = torch.rand((n, hd // 2, 2), generator=g).cuda()
    slots = torch.tensor([20, 21, 22, 40, 3], dtype=torch.int32, device="cuda")
    own = [torch.zeros((pages, kv, P, hd), dtype=torch.uint8, device="cuda"), torch.zeros((pages, kv, hd, P), dtype=torch.uint8, device="cuda"),
           torch.ones((pages, kv), device="cuda"), torch.ones((pages, kv), device="cuda")]
    q_out = torch.zeros((n, heads, hd), dtype=torch.bfloat16, device="cuda")
    pool = pages * kv * P * hd
    sizes = [2 * rows.numel(), 4 * table.numel(), 32, pool, pool, 32, 32, 2 * q_out.numel()]
    whole = torch.zeros(sum(sizes), dtype=torch.uint8, device="cuda")
    at = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    part = lambda i, t, shape: whole[at[i]:at[i + 1]].view(t)[:torch.Size(shape).numel()].view(shape)  # noqa: E731
    r, tb, sl = part(0, torch.bfloat16, rows.shape), part(1, torch.float32, table.shape), part(2, torch.int32, (n,))
    mine = [part(3, torch.uint8, own[0].shape), part(4, torch.uint8, own[1].shape), part(5, torch.float32, own[2].shape),
            part(6, torch.float32, own[3].shape)]
    qo = part(7, torch.bfloat16, q_out.shape)
    for a, b in ((r, rows), (tb, table), (sl, slots), (mine[2], own[2]), (mine[3], own[3])):
        a.copy_(b)
    hip.kv_store_rotary_paged(r[:, heads:heads + kv], r[:, heads + kv:], tb, sl, *mine, q=r[:, :heads], q_out=qo)
    hip.kv_store_rotary_paged(rows[:, heads:heads + kv], rows[:, heads + kv:], table, slots, *own, q=rows[:, :heads], q_out=q_out)
    assert torch.equal(qo, q_out) and all(torch.equal(a, b) for a, b in zip(mine, own)) and torch.equal(r, rows)
