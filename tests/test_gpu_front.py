"""The attention front of prompt chunks (q36_attn_front through attn_fused.attn_front) against the formula in 64 bits.

Bars, from the arithmetic: a value y is formed in fp32 (the sum of 256 squares, the root, two or three products and the
sum of two products: together below 2^-19 of the largest magnitude that enters, |y_i| + |y_{i+32}|) and rounded once: by
2^-8 of itself to bf16, by 2^-4 of itself, or 2^-10 where e4m3 is subnormal, to e4m3."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D, ROWS, EPS, MAX_POS = 16, 2, 256, 9216, 1e-6, 500


@pytest.fixture(scope="module")
def attn():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import attn_fused
    return attn_fused


def make(T, seed, dev, axes=1, scale=1.5, max_pos=MAX_POS):
    g = torch.Generator().manual_seed(seed)
    inv = 1e7 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv
    d = dict(qkv=(torch.randn((T, ROWS), generator=g) * scale).to(torch.bfloat16),
             qw=(torch.randn(D, generator=g) * 0.1).to(torch.bfloat16), kw=(torch.randn(D, generator=g) * 0.1).to(torch.bfloat16),
             cos_sin=torch.cat([ang.cos(), ang.sin()], 1).float(),
             pos=torch.randint(0, max_pos, (axes, T), generator=g, dtype=torch.int32),
             loc=torch.randperm(T + 9, generator=g)[:T])
    return {k: v.to(dev) for k, v in d.items()}


def formula(d, axis_of, max_pos=MAX_POS):
    """q, gate, k, v in 64 bits and the magnitudes that enter q and k."""
    x = d["qkv"].double()
    T = x.shape[0]
    qg, kv = x[:, :8192].reshape(T, HQ, 2, D), x[:, 8192:].reshape(T, 2, HKV, D)
    pair = torch.arange(32, device=x.device)
    at = d["pos"].long().clamp(0, max_pos - 1)[torch.tensor(axis_of, device=x.device)].t()
    c, s = d["cos_sin"].double()[at, pair][:, None], d["cos_sin"].double()[at, 32 + pair][:, None]
    out = []
    for h, w in ((qg[:, :, 0], d["qw"]), (kv[:, 0], d["kw"])):
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * (1 + w.double())
        a, b = y[..., :32], y[..., 32:64]
        mag = y.abs()
        pairs = a.abs() + b.abs()
        out.append((torch.cat([a * c - b * s, b * c + a * s, y[..., 64:]], -1), torch.cat([pairs, pairs, mag[..., 64:]], -1)))
    return out[0], qg[:, :, 1], out[1], kv[:, 1]


def near(got, want, mag, e4m3, what):
    want = want.clamp(-448, 448) if e4m3 else want
    step = torch.maximum(want.abs() * 2**-4, torch.full_like(want, 2**-10)) if e4m3 else want.abs() * 2**-8
    bound = step + mag * 2**-19
    off = (got.double() - want).abs()
    worst = float((off / bound).nan_to_num(posinf=0).max()) if off.numel() else 0.0
    print(f"{what}: {worst:.3f} of the bar", flush=True)
    assert bool((off <= bound).all()), f"{what}: {worst} of the bar"


def value(codes):
    return codes.view(torch.float8_e4m3fn).float()


def check(attn, d, dev, axes, q8, what, max_pos=MAX_POS, cache=True):
    T = d["qkv"].shape[0]
    kc, vc = (torch.full((T + 9, HKV, D), 0x55, dtype=torch.uint8, device=dev) for _ in range(2))
    q, gate = attn.attn_front(d["qkv"], d["qw"], d["kw"], EPS, d["cos_sin"], d["pos"] if axes else d["pos"][0],
                              cache=(kc, vc, d["loc"]) if cache else None, axes=axes,
                              q_dtype=torch.uint8 if q8 else torch.bfloat16)
    torch.cuda.synchronize()
    (wq, mq), wg, (wk, mk), wv = formula(d, axes.axis_of if axes else [0] * 32, max_pos)
    near(value(q) if q8 else q, wq, mq, q8, f"{what} q")
    assert torch.equal(gate.double(), wg)
    ok = (d["loc"] >= 0) & (d["loc"] < T + 9)
    if cache:
        at = d["loc"][ok]
        near(value(kc[at]), wk[ok], mk[ok], True, f"{what} k")
        near(value(vc[at]), wv[ok], wv[ok].abs() * 0, True, f"{what} v")
        rest = torch.ones(T + 9, dtype=torch.bool, device=dev)
        rest[at] = False
        assert bool((kc[rest] == 0x55).all()) and bool((vc[rest] == 0x55).all())
    return q, gate, kc, vc


AXES = {"one": None, "sections": ((11, 11, 10), False), "woven": ((11, 11, 10), True), "two": ((20, 12), False),
        "four": ((8, 8, 8, 8), True), "height": ((0, 32), False), "skewed": ((31, 0, 1), True)}


@pytest.mark.parametrize("kind", sorted(AXES))
@pytest.mark.parametrize("q8", [False, True])
def test_front_is_the_formula(attn, dev, kind, q8):
    axes = None if AXES[kind] is None else attn.RopeAxes(*AXES[kind])
    for T in (1, 3, 17, 130):
        print(f"front {kind} q8={q8} T={T}", flush=True)
        check(attn, make(T, T + 31 * q8, dev, axes.axes if axes else 1), dev, axes, q8, f"T={T}")


def test_axes_of_the_pairs(attn):
    assert attn.RopeAxes((11, 11, 10)).axis_of == [0] * 11 + [1] * 11 + [2] * 10
    woven = attn.RopeAxes((11, 11, 10), True).axis_of
    assert woven[:6] == [0, 1, 2, 0, 1, 2] and woven.count(1) == 11 and woven.count(2) == 10 and woven[31] == 1 and woven[30] == 0


def test_axes_that_agree_are_one_axis(attn, dev):
    """Positions alike on all axes give the bits of one axis."""
    d = make(37, 5, dev, 3)
    d["pos"][:] = d["pos"][0].clone()
    one = attn.attn_front(d["qkv"], d["qw"], d["kw"], EPS, d["cos_sin"], d["pos"][0].contiguous())
    three = attn.attn_front(d["qkv"], d["qw"], d["kw"], EPS, d["cos_sin"], d["pos"], axes=attn.RopeAxes((11, 11, 10), True))
    torch.cuda.synchronize()
    assert torch.equal(one[0], three[0]) and torch.equal(one[1], three[1])


def test_rows_without_a_slot_and_positions_outside(attn, dev):
    d = make(40, 6, dev, 3)
    d["loc"][5], d["loc"][6], d["loc"][7] = -1, 49, 2**40
    d["pos"][0, 3], d["pos"][1, 4], d["pos"][2, 9] = -7, MAX_POS, 2**31 - 1
    check(attn, d, dev, attn.RopeAxes((11, 11, 10)), True, "outside")


def test_strided_rows_and_no_cache(attn, dev):
    d = make(21, 7, dev)
    wide = torch.zeros((21, ROWS + 64), dtype=torch.bfloat16, device=dev)
    wide[:, :ROWS] = d["qkv"]
    a = check(attn, d, dev, None, False, "straight")
    b = check(attn, {**d, "qkv": wide[:, :ROWS]}, dev, None, False, "strided")
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])
    check(attn, d, dev, None, True, "no cache", cache=False)
    pos = torch.zeros((3, 30), dtype=torch.int32, device=dev)  # positions of a longer batch: a row stride
    pos[:, :21] = d["pos"][0]
    s = attn.attn_front(d["qkv"], d["qw"], d["kw"], EPS, d["cos_sin"], pos[:, :21], axes=attn.RopeAxes((11, 11, 10)))
    torch.cuda.synchronize()
    assert torch.equal(s[0], a[0])


def test_values_at_the_borders(attn, dev):
    """Zero rows, values past e4m3's largest, NaN and infinity: where they are, and nowhere else."""
    d = make(6, 8, dev)
    d["qkv"][0] = 0
    d["qkv"][1, 8704:] = 1000.0
    d["qkv"][1, 8704] = -1000.0
    kc, vc = (torch.zeros((6, HKV, D), dtype=torch.uint8, device=dev) for _ in range(2))
    d["qkv"][3, 3 * 512 + 100] = float("nan")   # a value of q head 3
    d["qkv"][4, 8704 + 256 + 7] = float("nan")  # a value of v head 1
    d["qkv"][5, 2 * 512 + 256 + 9] = float("inf")  # a gate
    loc = torch.arange(6, device=dev)
    q, gate = attn.attn_front(d["qkv"], d["qw"], d["kw"], EPS, d["cos_sin"], d["pos"][0], cache=(kc, vc, loc), q_dtype=torch.uint8)
    torch.cuda.synchronize()
    q, k, v = value(q), value(kc), value(vc)
    assert bool((q[0] == 0).all()) and bool((k[0] == 0).all())
    assert bool((v[1].flatten()[1:] == 448).all()) and float(v[1, 0, 0]) == -448
    bad = torch.isnan(q)
    assert bool(bad[3, 3].all()) and int(bad.sum()) == D
    assert not bool(torch.isnan(k).any())
    assert torch.isnan(v).nonzero().tolist() == [[4, 1, 7]]
    assert torch.isinf(gate).nonzero().tolist() == [[5, 2, 9]]


def test_no_tokens(attn, dev):
    d = make(0, 9, dev)
    q, gate = attn.attn_front(d["qkv"], d["qw"], d["kw"], EPS, d["cos_sin"], d["pos"][0])
    assert q.shape == (0, HQ, D) and gate.shape == (0, HQ, D)


def test_close_to_the_projection_entry(attn, dev):
    """The front over projected rows against attn_proj, which rounds to bf16 between its steps: three roundings of 2^-8
    apart at most (the norm's, the rotation's products of them, the output's)."""
    from bundles_amd import synth
    from bundles_amd.qwen36_layer import glue
    T = 150
    ai = synth.attn_inputs(T, dev, seed=3)
    w = attn.prepare_weights(ai["wqg"], ai["wk"], ai["wv"], ai["wo"])
    cs = attn.rope_cos_sin(MAX_POS, device=dev)
    pos = torch.arange(20, 20 + T, dtype=torch.int32, device=dev)
    kc, vc = (torch.zeros((T, HKV, D), dtype=torch.uint8, device=dev) for _ in range(2))
    p = attn.attn_proj(ai["x"], w, ai["q_norm_w"], ai["k_norm_w"], EPS, cs, pos, attn.Workspace(T, dev))
    qkv = torch.empty((T, ROWS), dtype=torch.bfloat16, device=dev)
    fw = glue.prepare_fp8_weight(torch.cat([ai["wqg"], ai["wk"], ai["wv"]]))
    glue.fp8_linear(ai["x"], fw, glue.LinearWorkspace(T, 2048, dev), segments=[(0, qkv)])
    q, gate = attn.attn_front(qkv, ai["q_norm_w"], ai["k_norm_w"], EPS, cs, pos, cache=(kc, vc, torch.arange(T, device=dev)))
    torch.cuda.synchronize()
    assert torch.equal(gate, p["gate"])
    assert torch.equal(vc, p["v8"])
    (_, mq), _, _, _ = formula(dict(qkv=qkv, qw=ai["q_norm_w"], kw=ai["k_norm_w"], cos_sin=cs, pos=pos[None]), [0] * 32)
    assert bool(((q.double() - p["q"].double()).abs() <= 3 * 2**-8 * mq).all())


def test_front_replays(attn, dev):
    d = make(64, 10, dev, 3)
    axes = attn.RopeAxes((11, 11, 10), True)
    kc, vc = (torch.zeros((73, HKV, D), dtype=torch.uint8, device=dev) for _ in range(2))
    q, gate = (torch.empty((64, HQ, D), dtype=t, device=dev) for t in (torch.uint8, torch.bfloat16))
    call = lambda: attn.attn_front(d["qkv"], d["qw"], d["kw"], EPS, d["cos_sin"], d["pos"], cache=(kc, vc, d["loc"]),  # noqa: E731
                                   axes=axes, q_dtype=torch.uint8, q=q, gate=gate)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(3):
        e = make(64, 20 + seed, dev, 3)
        for k in d:
            d[k].copy_(e[k])
        call()
        torch.cuda.synchronize()
        want = [t.clone() for t in (q, gate, kc, vc)]
        for t in (q, gate):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((q, gate, kc, vc), want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
