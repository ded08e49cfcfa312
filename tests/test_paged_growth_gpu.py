"""Single tokens whose page moves to a larger scale: a decode step that appends one
token to each request, the value that needs the larger scale among it.  What is stored is
compared byte for byte with the definition; how long it takes, with a run of two."""
import time

import pytest

from test_paged_gpu import DTYPES, _store, store_reference

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("P,hd", [(16, 16), (16, 256), (32, 80), (64, 64), (64, 128), (128, 112), (128, 128), (256, 64), (256, 256)])
def test_growing_pages(torch, hip, dtype, P, hd):
    """Places from the first to the last; of each page and head keys, values, both or neither grow."""
    kv, g = 4, torch.Generator().manual_seed(P + hd)
    places = sorted({0, 1, 2, 3, 4, 7, 14, 15, P // 2, P // 2 + 1, P - 2, P - 1} & set(range(P)))
    pages = torch.randperm(len(places), generator=g).tolist()
    slots = [p * P + at for p, at in zip(pages, places)]
    rows = torch.randn((len(slots), 2, kv, hd), generator=g)
    # head 0: neither, 1: keys, 2: values, 3: both, 16, 128 or 4096 times as large
    by = torch.tensor([2.0, 16.0, 512.0])[torch.randint(0, 3, (len(slots), 1), generator=g)]
    rows[:, 0, 1::2] *= 8 * by[..., None]
    rows[:, 1, 2:] *= 8 * by[..., None]
    rows = rows.to(getattr(torch, dtype)).cuda()
    n = len(places)
    cache = [torch.randn((n, kv, P, hd), generator=g).mul(60).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]
    for c in cache:  # (marks of what was not finite stay)
        c.view(-1)[torch.randint(0, c.numel(), (c.numel() // 50,), generator=g)] = 0x7f
        c.view(-1)[torch.randint(0, c.numel(), (c.numel() // 50,), generator=g)] = 0xff
    scales = [torch.full((n, kv), 2.0 ** -6) for _ in range(2)]
    print(f"growing {dtype} P {P} hd {hd}", flush=True)
    _, _, ks, vs = _store(torch, hip, (rows[:, 0], rows[:, 1]), slots, cache, scales, P)
    behind = [p for p, at in zip(pages, places) if at > 0]
    assert (ks.cpu()[behind][:, [0, 2]] == 2.0 ** -6).all() and (ks.cpu()[behind][:, [1, 3]] > 2.0 ** -6).all()
    assert (vs.cpu()[behind][:, [0, 1]] == 2.0 ** -6).all() and (vs.cpu()[behind][:, [2, 3]] > 2.0 ** -6).all()


def test_a_decode_that_grows(torch, hip):
    """Token after token into the same pages, each larger than those before, rotated and not: what
    one call for each page's first half and one token a call give is what the definition gives."""
    B, P, kv, hd = 5, 32, 2, 64
    rows = torch.randn((P, B, 2, kv, hd), generator=torch.Generator().manual_seed(3))
    rows *= torch.exp2(torch.arange(P) * 0.7)[:, None, None, None, None]
    rows = rows.cuda()
    table = torch.zeros((B, hd // 2, 2), device="cuda")
    table[..., 0] = 1.0  # (angles of zero: the same keys)
    empty = [torch.zeros((B, kv, P, hd), dtype=torch.uint8) for _ in range(2)]
    plain = [empty[0].cuda(), empty[1].transpose(2, 3).contiguous().cuda(), torch.ones((B, kv), device="cuda"), torch.ones((B, kv), device="cuda")]
    turned = [t.clone() for t in plain]
    want = [(empty[i].clone(), torch.ones((B, kv))) for i in range(2)]
    for at in range(P):
        slots = [b * P + at for b in range(B)]
        sl = torch.tensor(slots, dtype=torch.int32, device="cuda")
        x = rows[at]
        hip.kv_store_paged(x[:, 0], x[:, 1], sl, *plain)
        hip.kv_store_rotary_paged(x[:, 0], x[:, 1], table, sl, *turned)
        for i in range(2):
            w, s = store_reference(torch, x[:, i].double().cpu(), slots, *want[i], P, False)
            want[i] = (w, s.float())
    assert torch.equal(plain[0].cpu(), want[0][0]) and torch.equal(plain[1].transpose(2, 3).cpu(), want[1][0])
    assert torch.equal(plain[2].cpu(), want[0][1]) and torch.equal(plain[3].cpu(), want[1][1])
    for a, b in zip(plain, turned):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rotated", [False, True])
def test_a_single_token_moves_its_page_as_fast_as_two(torch, hip, rotated):
    """Both move the page's earlier tokens, two by a whole workgroup; a token alone has less to do
    otherwise (by one wave that waited for every piece it took 1.5 times as long as two)."""
    B, kv, P, hd, n = 64, 8, 256, 256, 16
    cache = [torch.randint(0, 120, s, dtype=torch.uint8, device="cuda") for s in ((B, kv, P, hd), (B, kv, hd, P))]
    scales = [torch.ones((B, kv), device="cuda") for _ in range(2)]
    rows = torch.randn((2 * B, 2, kv, hd), device="cuda").bfloat16()
    table = torch.rand((2 * B, hd // 2, 2), device="cuda")
    least = {}
    for tokens in (1, 2):
        at = torch.arange(B)[:, None] * P + P - tokens + torch.arange(tokens)[None]
        slots, x = at.reshape(-1).int().cuda(), rows[:tokens * B]

        def step():
            for s in scales:
                s.fill_(2.0 ** -12)
            if rotated:
                hip.kv_store_rotary_paged(x[:, 0], x[:, 1], table[:tokens * B], slots, *cache, *scales)
            else:
                hip.kv_store_paged(x[:, 0], x[:, 1], slots, *cache, *scales)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(n):
                step()
        took = []
        for _ in range(12):
            torch.cuda.synchronize()
            start = time.perf_counter()
            graph.replay()
            torch.cuda.synchronize()
            took.append(time.perf_counter() - start)
        least[tokens] = min(took[2:])
    print("one token %.1f us, two %.1f" % (least[1] / n * 1e6, least[2] / n * 1e6), flush=True)
    assert least[1] <= 1.3 * least[2], least
