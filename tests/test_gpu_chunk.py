"""The chunk attention (q36_attn_chunk through attn_fused.attn_chunk) against the formula in 64 bits.

Bar for each output, from the arithmetic (v the values, p the softmax weights of the formula, l = sum exp(s - max)):
  2^-8 |o|                       the output's rounding to bf16
  2^-11 sum p |v|                each weight's rounding to f16 ...
  2^-25 sum |v| / l              ... or, below f16's normal range, its absolute half step
  2 d sum p |v|                  the scores' error d: 256 products of e4m3 values added in fp32, each sum within 2^-23 of
                                 the magnitudes so far, so d = 2^-15 scale max_j sum_i |q_i k_i|
  2^-15 sum p |v|                exp2 (an ulp), sums of weights and outputs in fp32 over up to 2^8 partial sums
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D, G = 16, 2, 256, 8
SCALE = 1.0 / 16.0


@pytest.fixture(scope="module")
def attn():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import attn_fused
    return attn_fused


def codes(t):
    return t.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def value(c):
    return c.view(torch.float8_e4m3fn).double()


def make(lens, P, seed, dev, q8=True, qscale=1.2, lead=0, tail=0, extra=1):
    """Requests of (new, keys) with distinct pages in random order; lead / tail rows of q that belong to no request."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-k // P) for _, k in lens]
    total = sum(pages) + 3
    perm = torch.randperm(total, generator=g).to(torch.int32)
    pt = torch.zeros((len(lens), max(pages + [1]) + extra), dtype=torch.int32)
    o = 0
    for b, n in enumerate(pages):
        pt[b, :n] = perm[o:o + n]
        o += n
    n = torch.tensor([a for a, _ in lens])
    qsl = lead + torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)])
    T = lead + int(n.sum()) + tail
    gd = torch.Generator(device=dev).manual_seed(seed)
    head = 0.5 + 1.5 * torch.rand((1, HKV, 1), generator=gd, device=dev)
    kc, vc = (codes(torch.randn((total * P, HKV, D), generator=gd, device=dev) * head) for _ in range(2))
    q = (torch.randn((T, HQ, D), generator=gd, device=dev) * qscale).to(torch.bfloat16)
    return dict(q=codes(q.float()) if q8 else q, kc=kc, vc=vc, pt=pt.to(dev), P=P, lens=lens,
                seqlens=torch.tensor([k for _, k in lens], dtype=torch.int32, device=dev), qsl=qsl.to(torch.int32).to(dev))


def formula(h):
    """The output in 64 bits, its bar, and the rows that belong to a request."""
    q = value(h["q"]) if h["q"].dtype == torch.uint8 else value(codes(h["q"].float()))
    out, bar = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mine = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    qsl, P = h["qsl"].tolist(), h["P"]
    for b, (n, L) in enumerate(h["lens"]):
        mine[qsl[b]:qsl[b + 1]] = True
        if L == 0 or n == 0:
            continue
        key = torch.arange(L, device=q.device)
        slot = h["pt"][b, key // P].long() * P + key % P
        k, v = value(h["kc"][slot]), value(h["vc"][slot])
        for a in range(qsl[b], qsl[b + 1], 512):
            e = min(a + 512, qsl[b + 1])
            hide = key[None, :] > (L - n + torch.arange(a - qsl[b], e - qsl[b], device=q.device))[:, None]
            for hh in range(HQ):
                kk, vv, qq = k[:, hh // G], v[:, hh // G], q[a:e, hh]
                s = (qq @ kk.t().contiguous()) * SCALE
                s = s.masked_fill(hide, -torch.inf)
                top = s.amax(1, keepdim=True)
                x = torch.where(hide, 0.0, torch.exp(s - top.nan_to_num(neginf=0.0)))
                l = x.sum(1, keepdim=True)  # noqa: E741
                seen = l > 0
                p = x / torch.where(seen, l, 1.0)
                o, absv = p @ vv, vv.abs()
                pv = p @ absv
                d = 2**-15 * SCALE * (qq.abs() @ kk.abs().t().contiguous()).masked_fill(hide, 0).amax(1, keepdim=True)
                flush = ((~hide).double() @ absv) * 2**-25 / torch.where(seen, l, 1.0)
                out[a:e, hh] = o
                bar[a:e, hh] = 2**-8 * o.abs() + (2**-11 + 2**-15 + 2 * d) * pv + flush
    return out, bar, mine


def run(attn, h, dev, ws=None, out=None):
    ws = attn.ChunkWorkspace(dev) if ws is None else ws
    return attn.attn_chunk(h["q"], h["kc"], h["vc"], h["pt"], h["seqlens"], h["qsl"], SCALE, ws, page_size=h["P"], out=out)


def check(attn, h, dev, what, ws=None):
    print(f"chunk {what}", flush=True)
    out = torch.full(h["q"].shape, 77.0, dtype=torch.bfloat16, device=dev)
    run(attn, h, dev, ws, out)
    torch.cuda.synchronize()
    want, bar, mine = formula(h)
    assert bool((out[~mine] == 77).all()), f"{what}: rows of no request written"
    off = (out.double() - want).abs()[mine]
    worst = float((off / bar[mine].clamp(min=1e-300)).max()) if off.numel() else 0.0
    rel = float(off.norm() / want[mine].norm().clamp(min=1e-300)) if off.numel() else 0.0
    print(f"chunk {what}: {worst:.3f} of the bar, relative {rel:.2e}", flush=True)
    assert bool(torch.isfinite(out[mine]).all()) and bool((off <= bar[mine]).all()), f"{what}: {worst} of the bar"
    return out


LENS = {
    "one token": [(1, 1)],
    "short": [(5, 300)],
    "tile borders": [(1, 32), (1, 33), (4, 31), (5, 64), (8, 8), (9, 41), (16, 16), (17, 17), (31, 64), (32, 32), (33, 97), (64, 64), (65, 200)],
    "empty requests": [(0, 0), (3, 9), (0, 50), (40, 40), (0, 0), (1, 700)],
    "prompt": [(500, 500)],
    "chunk behind a prefix": [(210, 1000)],
    "few rows, long": [(7, 9001)],
    "one row, long": [(1, 20011)],
    "mixed": [(1, 900), (130, 2000), (1, 33), (2, 5000), (61, 61), (1, 1), (300, 301), (12, 700)],
    "decoding batch": [(1, 37 * b % 1500 + 1) for b in range(70)],
}


@pytest.mark.parametrize("name", sorted(LENS))
@pytest.mark.parametrize("P,q8", [(1, True), (16, False), (64, True)])
def test_chunk_is_the_formula(attn, dev, name, P, q8):
    h = make(LENS[name], P, len(name) + P, dev, q8)
    check(attn, h, dev, f"{name} P={P} q8={q8}")


def test_many_requests(attn, dev):
    check(attn, make([(b % 3, b % 90 + 3) for b in range(701)], 8, 3, dev), dev, "701 requests")


def test_large_chunk(attn, dev):
    check(attn, make([(2048, 2500), (1000, 1000)], 16, 4, dev), dev, "2048 + 1000")


def test_peaked_and_flat_softmax(attn, dev):
    """Scores that span many binades (the running maximum grows through the keys), and queries of zero."""
    check(attn, make([(40, 3000), (3, 2000)], 1, 5, dev, qscale=6.0), dev, "peaked")
    h = make([(40, 900), (2, 1200)], 1, 6, dev)
    h["kc"][:] = h["kc"][h["pt"][0, 0].long()].clone()
    h["q"][:] = 0
    check(attn, h, dev, "flat")


def test_growing_maximum(attn, dev):
    """Each later key scores higher than all before it, by far: every step rescales."""
    h = make([(33, 800)], 1, 7, dev)
    k = torch.linspace(-8, 8, 800, device=dev)[:, None, None].expand(800, HKV, D)
    h["kc"][h["pt"][0, :800].long()] = codes(k)
    h["q"][:] = codes(torch.full((33, HQ, D), 1.5, device=dev))
    check(attn, h, dev, "growing maximum")


def test_rows_of_no_request_are_left(attn, dev):
    check(attn, make([(9, 100), (0, 4), (35, 50)], 1, 8, dev, lead=6, tail=29), dev, "lead and tail")


def test_rows_that_see_no_key_are_zero(attn, dev):
    h = make([(6, 6), (40, 40), (3, 8)], 4, 9, dev)
    h["seqlens"][0], h["seqlens"][1], h["seqlens"][2] = 2, 5, 0
    h["lens"] = [(6, 2), (40, 5), (3, 0)]
    out = check(attn, h, dev, "fewer keys than new tokens")
    assert bool((out[:4] == 0).all()) and bool((out[6:41] == 0).all()) and bool((out[46:] == 0).all())
    assert bool((out[4:6] != 0).any()) and bool((out[41:46] != 0).any())


def test_shared_pages(attn, dev):
    """Requests that share a prefix's pages."""
    h = make([(20, 500), (20, 500), (1, 500)], 16, 10, dev)
    h["pt"][1, :20] = h["pt"][0, :20]
    h["pt"][2] = h["pt"][0]
    check(attn, h, dev, "shared pages")


def test_results_repeat(attn, dev):
    ws = attn.ChunkWorkspace(dev)
    h = make([(70, 5000), (1, 9000), (300, 400)], 1, 11, dev)
    first = run(attn, h, dev, ws).clone()
    other = make([(500, 700), (3, 3)], 1, 12, dev)
    run(attn, other, dev, ws)
    assert torch.equal(run(attn, h, dev, ws), first)


def test_a_cache_past_32_bits(attn, dev):
    """Slots whose byte offsets pass 2^31 and 2^32."""
    slots = (1 << 23) + 4096
    h = make([(37, 600), (2, 900)], 16, 13, dev)
    small = h["kc"].shape[0]
    pages = torch.randperm(slots // 16, generator=torch.Generator().manual_seed(1))[:small // 16]
    pages[:4] = torch.tensor([slots // 16 - 1, slots // 16 - 2, (1 << 22) // 16, (1 << 23) // 16])
    kc, vc = (torch.zeros((slots, HKV, D), dtype=torch.uint8, device=dev) for _ in range(2))
    at = (pages[:, None] * 16 + torch.arange(16)).reshape(-1).to(dev)
    assert at.unique().numel() == small
    kc[at], vc[at] = h["kc"][:small], h["vc"][:small]
    want, bar, _ = formula(h)
    out = attn.attn_chunk(h["q"], kc, vc, pages.to(torch.int32).to(dev)[h["pt"].long()].contiguous(), h["seqlens"], h["qsl"], SCALE,
                          attn.ChunkWorkspace(dev), page_size=16)
    torch.cuda.synchronize()
    assert bool(((out.double() - want).abs() <= bar).all())


def test_what_a_row_does_not_see_does_not_reach_it(attn, dev):
    """NaN keys and values: later new tokens' and unused slots' leave a row alone, seen ones make it NaN."""
    NAN = 0x7F
    for n, L in ((40, 200), (6, 50), (100, 100), (3, 4000)):
        h = make([(n, L)], 1, 14 + n, dev)
        clean, bar, _ = formula(h)
        used = torch.zeros(h["kc"].shape[0], dtype=torch.bool, device=dev)
        used[h["pt"][0, :L].long()] = True
        h["kc"][~used] = NAN
        h["vc"][~used] = NAN
        h["pt"][0, L:] = int((~used).nonzero()[0])
        first = n - 2  # the new token whose value, and the one after whose key, is NaN
        h["vc"][h["pt"][0, L - n + first].long(), 1, 17] = NAN
        h["kc"][h["pt"][0, L - 1].long(), 0, 5] = 0xFF
        out = run(attn, h, dev)
        torch.cuda.synchronize()
        off = (out.double() - clean).abs()
        print(f"NaN n={n} L={L}", flush=True)
        assert bool((off[:first] <= bar[:first]).all())
        nan = torch.isnan(out)
        want = torch.zeros_like(nan)
        want[first:, G:, 17] = True
        want[n - 1, :G] = True
        assert torch.equal(nan, want)
        keep = ~want
        assert bool((off[keep] <= bar[keep]).all())


def test_device_data_out_of_range_stay_inside(attn, dev):
    """Tables, lengths and starts that point outside: the calls end, and requests that are in order are served."""
    h = make([(30, 300), (5, 40), (3, 90)], 1, 15, dev)
    want, bar, _ = formula(h)
    h["pt"][1, :20] = torch.tensor([-1, 2**31 - 1, -2**31, h["kc"].shape[0]] * 5, dtype=torch.int32, device=dev)
    out = run(attn, h, dev).double()
    torch.cuda.synchronize()
    for a, e in ((0, 30), (35, 38)):
        assert bool(((out[a:e] - want[a:e]).abs() <= bar[a:e]).all())
    for lens in ([2**31 - 1, 40, 90], [-5, 40, 90]):
        h2 = dict(h, seqlens=torch.tensor(lens, dtype=torch.int32, device=dev))
        out = run(attn, h2, dev).double()
        torch.cuda.synchronize()
        assert bool(((out[35:] - want[35:]).abs() <= bar[35:]).all())
    for qsl in ([0, 2**31 - 1, 35, 38], [-9, 30, 35, 10**6], [38, 0, 38, 0]):
        run(attn, dict(h, qsl=torch.tensor(qsl, dtype=torch.int32, device=dev)), dev)
        torch.cuda.synchronize()


def test_two_streams(attn, dev):
    jobs = [make([(70, 3000), (1, 500)], 1, 16, dev), make([(5, 8000), (200, 200)], 16, 17, dev)]
    alone = [run(attn, h, dev).clone() for h in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    spaces = [attn.ChunkWorkspace(dev) for _ in jobs]
    outs = [[torch.empty_like(a) for _ in range(3)] for a in alone]
    torch.cuda.synchronize()
    for r in range(3):
        for h, s, w, o in zip(jobs, streams, spaces, outs):
            attn.attn_chunk(h["q"], h["kc"], h["vc"], h["pt"], h["seqlens"], h["qsl"], SCALE, w, page_size=h["P"], out=o[r], stream=s)
    torch.cuda.synchronize()
    for o, a in zip(outs, alone):
        for x in o:
            assert torch.equal(x, a)


def test_replays_follow_the_lengths(attn, dev):
    """One captured call, padded to 90 rows and 4 requests, over other lengths at each replay; two graphs share a workspace."""
    P, T, B = 4, 90, 4
    ws = attn.ChunkWorkspace(dev)
    h = make([(20, 700)] * B, P, 18, dev, tail=10)
    out = torch.empty((T, HQ, D), dtype=torch.bfloat16, device=dev)
    other = make([(100, 150)], 1, 19, dev)
    oout = torch.empty((100, HQ, D), dtype=torch.bfloat16, device=dev)
    want_other = run(attn, other, dev).clone()
    call = lambda: run(attn, h, dev, ws, out)  # noqa: E731
    call()
    run(attn, other, dev, ws, oout)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        call()
    with torch.cuda.graph(g2):
        run(attn, other, dev, ws, oout)
    for lens in ([(1, 1), (1, 700), (0, 0), (1, 33)], [(60, 700), (0, 9), (5, 5), (20, 650)], [(1, 600)] * 4, [(90, 90), (0, 0), (0, 0), (0, 0)]):
        n = torch.tensor([a for a, _ in lens])
        h["lens"] = lens
        h["qsl"].copy_(torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]).to(torch.int32))
        h["seqlens"].copy_(torch.tensor([k for _, k in lens], dtype=torch.int32))
        out.fill_(77)
        oout.zero_()
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        want, bar, mine = formula(h)
        off = (out.double() - want).abs()
        assert bool((off[mine] <= bar[mine]).all()) and bool((out[~mine] == 77).all())
        assert torch.equal(oout, want_other)
        call()
        torch.cuda.synchronize()


def test_a_chunk_is_its_tokens_one_by_one(attn, dev):
    """The chunk against decode attention of the same tokens, each with its own key count (its weights and sums are split
    otherwise, so each is within its bar of the formula)."""
    h = make([(6, 500)], 1, 20, dev, q8=False)
    want, bar, _ = formula(h)
    ws = attn.DecodeWorkspace(6, dev)
    one = attn.attn_decode(h["q"], h["kc"], h["vc"], h["pt"].repeat(6, 1).contiguous(),
                           torch.arange(495, 501, dtype=torch.int32, device=dev), 1, SCALE, ws)
    out = run(attn, h, dev)
    torch.cuda.synchronize()
    assert bool(((out.double() - one.double()).abs() <= 2 * bar).all())


def test_no_tokens(attn, dev):
    h = make([(0, 5)], 1, 21, dev)
    assert run(attn, h, dev).shape == (0, HQ, D)


def test_row_starts_that_overlap_past_what_a_call_deals(attn, dev):
    """Row starts that count every row for every second request: their weights' sum passes 2^31 on the device, where the
    call's sizes alone do not.  Nothing is dealt, nothing is written, and the workspace serves the next call."""
    B, T, P, width = 64, 1 << 15, 1024, 8192
    ws = attn.ChunkWorkspace(dev)
    kc, vc = (torch.zeros((P, HKV, D), dtype=torch.uint8, device=dev) for _ in range(2))
    out = torch.full((T, HQ, D), 77.0, dtype=torch.bfloat16, device=dev)
    qsl = torch.tensor([0, T] * (B // 2) + [0], dtype=torch.int32, device=dev)
    attn.attn_chunk(torch.zeros((T, HQ, D), dtype=torch.uint8, device=dev), kc, vc, torch.zeros((B, width), dtype=torch.int32, device=dev),
                    torch.full((B,), P * width, dtype=torch.int32, device=dev), qsl, SCALE, ws, page_size=P, out=out)
    torch.cuda.synchronize()
    assert bool((out == 77).all())
    check(attn, make([(70, 900), (3, 40)], 16, 21, dev), dev, "after it", ws)


@pytest.mark.parametrize("lens", [[(40, 300)], [(5, 900), (1, 33)]], ids=["wide", "narrow"])
def test_queries_past_the_largest_code(attn, dev, lens):
    """bf16 queries are rounded to e4m3 with saturation: values past 448, infinities among them, count as 448, a NaN makes its
    row NaN, and the other rows of its wave keep their bits."""
    h = make(lens, 16, 22, dev, q8=False)
    plain = run(attn, h, dev).clone()
    q = h["q"]
    q[0, 3] = q[0, 3] * 100
    q[1, 9, 17], q[2, 0, 255], q[3, 15, 0] = 460.0, 465.0, -3.0e38
    q[2, 8, 100] = torch.inf
    q[4, 11, 64] = -torch.inf
    check(attn, h, dev, "saturated queries")
    q[1, 4, 5] = torch.nan
    out = run(attn, h, dev)
    torch.cuda.synchronize()
    assert bool(out[1, 4].isnan().all()) and int(out.isnan().any(-1).sum()) == 1
    touched = torch.zeros(out.shape[:2], dtype=torch.bool, device=dev)
    for t, hd in ((0, 3), (1, 9), (2, 0), (3, 15), (2, 8), (4, 11), (1, 4)):
        touched[t, hd] = True
    assert torch.equal(out[~touched], plain[~touched])


def test_a_workspace_may_hold_anything(attn, dev):
    """Memory of another use, made ready by the workspace entry, serves a call as fresh memory does; whatever is in the
    partials' part, and however many calls have passed."""
    from bundles_amd import _lib
    h = make([(300, 2000), (70, 900), (1, 5000)], 16, 23, dev)
    want = run(attn, h, dev).clone()
    for fill in (0xff, 0x00, 0x7f):
        ws = attn.ChunkWorkspace(dev)
        ws.buf.fill_(fill)
        _lib.check(_lib.lib().q36_attn_chunk_workspace_init(ws.buf.data_ptr(), ws.buf.numel(), _lib.stream_handle(None)), "init")
        for _ in range(3):
            out = run(attn, h, dev, ws)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("B,n,T", [(16384, 64, 1 << 20), (65535, 1, 65535), (65535, 3, (1 << 20) - 9)])
def test_the_largest_batches(attn, dev, B, n, T):
    """As many requests and rows as a call takes (outputs past 2^32 bytes): requests spread over the batch against the formula,
    and rows behind the last one left."""
    P, pages, width, keys = 64, 50, 2, 100
    g = torch.Generator(device=dev).manual_seed(24)
    kc, vc = (codes(torch.randn((pages * P, HKV, D), generator=g, device=dev)) for _ in range(2))
    q = torch.randint(0, 0x58, (T, HQ, D), generator=g, device=dev, dtype=torch.uint8)
    q[:, :, ::2] |= 0x80
    pt = torch.randint(0, pages, (B, width), generator=g, device=dev, dtype=torch.int32)
    seqlens = torch.full((B,), keys, dtype=torch.int32, device=dev)
    qsl = torch.arange(B + 1, device=dev, dtype=torch.int32) * n
    out = torch.full((T, HQ, D), 77.0, dtype=torch.bfloat16, device=dev)
    attn.attn_chunk(q, kc, vc, pt, seqlens, qsl, SCALE, attn.ChunkWorkspace(dev), page_size=P, out=out)
    torch.cuda.synchronize()
    assert bool((out[B * n:] == 77).all())
    for b in (0, 1, 511, 512, 513, B // 2, B - 2, B - 1):
        h = dict(q=q[b * n:(b + 1) * n], kc=kc, vc=vc, pt=pt[b:b + 1], P=P, lens=[(n, keys)], qsl=torch.tensor([0, n]))
        want, bar, _ = formula(h)
        off = (out[b * n:(b + 1) * n].double() - want).abs()
        assert bool((off <= bar).all()), f"request {b}: {float((off / bar).max())} of the bar"
