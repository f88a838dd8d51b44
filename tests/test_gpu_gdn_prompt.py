"""The recurrent layer's prompt (q36_gdn_prompt) against the recurrence in 64 bits, token by token.

Tolerances.  Output rows: one bf16 rounding (half a step, 2^-8 of the value at most) and the products behind it, whose
operands keep at least 11 significand bits in any kernel (half steps of 2^-12, two a product, one for an intermediate):
2^-8 + 2^-10 of the row's norm.  State: products of two operands of 22 bits (2^-22 with both roundings), sums of up to 128 + 64
terms in fp32 whose half steps (2^-24) add as their square root at random and cannot exceed 2^-24 (128 + 64) = 1.2e-5 of the sum
of magnitudes: 2e-5 of a head's largest value.  (Errors do not grow from chunk to chunk: the step S -> e^g S (1 - beta k k^T) is
a contraction.)  The conv state is copied: equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HK, HV, D, QKV = 16, 32, 128, 8192
OUT, STATE = 2.0 ** -8 + 2.0 ** -10, 2e-5


@pytest.fixture(scope="module")
def gdn():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import gdn_fused
    return gdn_fused


def inputs(lens, dev, seed, fresh=(), idx=torch.int64, rows=None, dt=torch.float32, pad=0):
    from bundles_amd import synth
    B, T = len(lens), sum(lens)
    rows = T if rows is None else rows
    f = synth.gdn_inputs(1, max(rows, 1), dev, seed=seed)
    g = torch.Generator().manual_seed(seed)
    slots = B + 3
    conv = torch.zeros((slots, QKV * 3 + pad), dtype=torch.bfloat16, device=dev)
    conv = torch.as_strided(conv, (slots, QKV, 3), (QKV * 3 + pad, 3, 1))
    conv.copy_(torch.randn((slots, QKV, 3), generator=g).to(dev))
    return dict(mixed=f["mixed"][:rows], z=f["z"][:rows], a=f["a"][:rows], b=f["b"][:rows], conv_state=conv, conv_w=f["conv_w"],
                A_log=f["A_log"], dt_bias=f["dt_bias"].to(dt),
                h0=(torch.randn((slots, HV, D, D), generator=g) * 0.1).to(dev),
                qsl=torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev),
                state_idx=torch.randperm(slots, generator=g)[:B].to(idx).to(dev), norm_w=f["norm_w"],
                prefix=torch.tensor([0 if r in fresh else 9 for r in range(B)], dtype=torch.int32, device=dev))


def plain(f, out=None, eps=1e-6, scale=D ** -0.5):
    """out, conv state and state in fp64, from the recurrence (on the GPU, one token of a request after another)."""
    rows = f["mixed"].shape[0]
    dev = f["mixed"].device
    o_all = torch.zeros((rows, HV * D), dtype=torch.float64, device=dev) if out is None else out.double()
    conv, h0 = f["conv_state"].double(), f["h0"].double()
    w = f["conv_w"].double()
    for r, si in enumerate(f["state_idx"].tolist()):
        lo, hi = (min(max(int(v), 0), rows) for v in f["qsl"][r:r + 2])
        if hi <= lo:
            continue
        if not 0 <= si < h0.shape[0]:
            o_all[lo:hi] = 0
            continue
        old = f["prefix"] is None or int(f["prefix"][r]) > 0
        S = h0[si].clone() if old else torch.zeros_like(h0[si])
        x = torch.cat([conv[si].t() if old else torch.zeros((3, QKV), dtype=torch.float64, device=dev), f["mixed"][lo:hi].double()])
        conv[si] = x[-3:].t()
        n = hi - lo
        y = sum(x[i:i + n] * w[:, i] for i in range(4))
        y = y / (1 + torch.exp(-y))
        q, k, v = y[:, :HK * D].view(n, HK, D), y[:, HK * D:2 * HK * D].view(n, HK, D), y[:, 2 * HK * D:].view(n, HV, D)
        q = (q / (q.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt() * scale).repeat_interleave(2, 1)
        k = (k / (k.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(2, 1)
        a = f["a"][lo:hi].double() + f["dt_bias"].double()
        e = torch.exp(-torch.exp(f["A_log"].double()) * torch.where(a > 30, a, torch.log1p(torch.exp(a.clamp(max=30)))))
        beta = torch.sigmoid(f["b"][lo:hi].double())
        o = torch.empty((n, HV, D), dtype=torch.float64, device=dev)
        for t in range(n):
            S *= e[t][:, None, None]
            u = beta[t][:, None] * (v[t] - (S * k[t][:, None, :]).sum(-1))
            S += u[:, :, None] * k[t][:, None, :]
            o[t] = (S * q[t][:, None, :]).sum(-1)
        h0[si] = S
        z = f["z"][lo:hi].double().view(n, HV, D)
        o = o / (o.pow(2).mean(-1, keepdim=True) + eps).sqrt() * f["norm_w"].double() * z / (1 + torch.exp(-z))
        o_all[lo:hi] = o.view(n, HV * D)
    return o_all, conv, h0


def call(gdn, f, ws=None, **kw):
    ws = ws or gdn.PromptWorkspace(f["mixed"].shape[0], len(f["state_idx"]), f["mixed"].device)
    return gdn.gdn_prompt(f["mixed"], f["z"], f["a"], f["b"], f["conv_state"], f["conv_w"], f["A_log"], f["dt_bias"], f["h0"],
                          f["qsl"], f["state_idx"], f["norm_w"], ws, prefix=f["prefix"], **kw)


def check(out, f, want, rows=None):
    o, conv, h0 = want
    assert torch.equal(f["conv_state"].double(), conv)
    got = out.double().view(-1, HV, D)
    ref = o.view(-1, HV, D)
    assert bool(torch.isfinite(got).all())
    err = ((got - ref).norm(dim=-1) - OUT * ref.norm(dim=-1)).max()
    rel = ((got - ref).norm(dim=-1) / (ref.norm(dim=-1) + 1e-30)).max()
    srel = ((f["h0"].double() - h0).abs().amax((-1, -2)) / (h0.abs().amax((-1, -2)) + 1e-30)).max()
    snorm = (f["h0"].double() - h0).norm() / h0.norm()
    print(f"worst row {float(rel):.2e}, state {float(srel):.2e} of a head's largest, norm {float(snorm):.2e}", flush=True)
    assert float(err) <= 0 and float(srel) <= STATE


@pytest.mark.parametrize("lens,fresh", [
    ([1], ()), ([1], (0,)), ([2, 1, 3], (1,)), ([7, 8, 9], (0, 2)), ([15, 16, 17], ()), ([31, 33, 32], (0,)),
    ([63, 64, 65], (1,)), ([127, 129], (0, 1)), ([200, 1, 0, 77, 5, 64], (0, 3)), ([517], (0,)), ([1, 300, 1, 1, 128], (1,))])
def test_prompt_lengths(gdn, dev, lens, fresh):
    print(f"prompt lens={lens} fresh={fresh}", flush=True)
    f = inputs(lens, dev, sum(lens) + len(lens), fresh)
    want = plain(f)
    check(call(gdn, f), f, want)


def test_prompt_continues_where_it_stopped(gdn, dev):
    """A prompt in pieces of odd lengths ends in the same state as in one piece, and every piece's rows are its own."""
    n, cuts = 400, [0, 1, 64, 130, 131, 200, 333, 400]
    f = inputs([n], dev, 5, (0,))
    whole = plain(f)
    outs = []
    for i, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])):
        p = dict(f, **{k: f[k][lo:hi].contiguous() for k in ("mixed", "z", "a", "b")})
        p["qsl"] = torch.tensor([0, hi - lo], dtype=torch.int32, device=dev)
        p["prefix"] = torch.tensor([lo], dtype=torch.int32, device=dev)
        outs.append(call(gdn, p))
    check(torch.cat(outs), f, whole)


def test_prompt_padded_batch_and_requests(gdn, dev):
    """Rows of no request stay as they were; a slot outside the pool zeroes its rows and writes nothing else."""
    f = inputs([40, 70, 3, 90], dev, 6, (3,), idx=torch.int32, rows=230, pad=8)
    f["state_idx"][1] = -1
    f["state_idx"][2] = 99
    out = torch.full((230, HV * D), 7.0, dtype=torch.bfloat16, device=dev)
    want = plain(f, out)
    call(gdn, f, out=out)
    check(out, f, want)
    assert bool((out[203:] == 7.0).all())


def test_prompt_rows_begin_behind_the_first(gdn, dev):
    f = inputs([50, 66], dev, 8, rows=140)
    f["qsl"] = torch.tensor([11, 61, 127], dtype=torch.int32, device=dev)
    out = torch.full((140, HV * D), -3.0, dtype=torch.bfloat16, device=dev)
    want = plain(f, out)
    call(gdn, f, out=out)
    check(out, f, want)
    assert bool((out[:11] == -3.0).all()) and bool((out[127:] == -3.0).all())


def test_prompt_fresh_requests_do_not_read_their_slots(gdn, dev):
    f = inputs([70, 2, 130], dev, 9, (0, 1))
    for r in (0, 1):
        f["h0"][f["state_idx"][r]] = float("nan")
        f["conv_state"][f["state_idx"][r]] = float("nan")
    used = f["state_idx"].tolist()
    want = plain(f)
    out = call(gdn, f)
    check(out, dict(f, conv_state=f["conv_state"][used], h0=f["h0"][used]), (want[0], want[1][used], want[2][used]))


@pytest.mark.parametrize("kind", ["strong", "none", "mixed", "tiny_beta", "same_key"])
def test_prompt_gates(gdn, dev, kind):
    """Decays that leave nothing of the state, none at all, one between gentle ones; a state of nearly one key."""
    f = inputs([140, 66], dev, 12, (0,))
    if kind == "strong":
        f["A_log"] = torch.full((HV,), 4.0, device=dev)
        f["a"].fill_(30.0)
    elif kind == "none":
        f["A_log"] = torch.full((HV,), -40.0, device=dev)
    elif kind == "mixed":  # a wall of forgetting, then slow decay: differences of large sums
        f["A_log"] = torch.full((HV,), 2.0, device=dev)
        f["a"].fill_(-6.0)
        f["a"][20:25] = 100.0
        f["a"][150] = 60.0
    elif kind == "tiny_beta":
        f["b"].fill_(-9.0)
        f["b"][::16] = 4.0
    else:
        f["mixed"][:, HK * D:2 * HK * D] = f["mixed"][3, HK * D:2 * HK * D]
        f["conv_w"][HK * D:2 * HK * D] = torch.tensor([0.0, 0.0, 0.0, 0.5])
        f["b"].fill_(3.0)
    want = plain(f)
    check(call(gdn, f), f, want)


@pytest.mark.parametrize("size", [1e-3, 300.0, 3e4])
def test_prompt_value_sizes(gdn, dev, size):
    """Values far from one: the state follows them whatever their size."""
    f = inputs([130, 20], dev, 13, (1,))
    f["mixed"][:, 2 * HK * D:] = (f["mixed"][:, 2 * HK * D:].float() * size).to(torch.bfloat16)
    f["mixed"][70:80, 2 * HK * D:] = (f["mixed"][70:80, 2 * HK * D:].float() * 1e-4).to(torch.bfloat16)
    want = plain(f)
    check(call(gdn, f), f, want)


def test_prompt_zero_rows(gdn, dev):
    """Rows of zeros: keys and queries of no length, no output."""
    f = inputs([90], dev, 14, (0,))
    f["mixed"][:20] = 0
    f["mixed"][50:60] = 0
    want = plain(f)
    out = call(gdn, f)
    check(out, f, want)
    assert not bool(out[:20].any())


def test_prompt_bf16_dt_bias_no_prefix_and_quantized_rows(gdn, dev):
    from bundles_amd.qwen36_layer.glue import linear_rows
    f = inputs([33, 100], dev, 15, dt=torch.bfloat16)
    f["prefix"] = None
    f["dt_bias"] = f["dt_bias"].contiguous()
    want = plain(f)
    oq = linear_rows(133, 4096, dev)
    out = call(gdn, f, oq=oq)
    check(out, f, want)
    y = out.float().view(-1, HV, D).cpu()  # (exact divisions)
    m = y.abs().amax(-1)
    assert bool((oq.scales.view(-1, HV).cpu() == m / 448).all())
    inv = torch.where(m > 0, torch.full_like(m, 448) / m, torch.zeros_like(m))  # (448 / m is a reciprocal times 448)
    codes = (y * inv[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert bool((oq.codes.view(torch.uint8).view(-1, HV, D).cpu() == codes.view(torch.uint8)).all())


def test_prompt_long(gdn, dev):
    f = inputs([2100, 40], dev, 16, (0,))
    want = plain(f)
    check(call(gdn, f), f, want)


def test_prompt_many_requests(gdn, dev):
    lens = [1 + (37 * i) % 23 for i in range(70)]
    f = inputs(lens, dev, 17, tuple(range(0, 70, 4)))
    want = plain(f)
    check(call(gdn, f), f, want)


def test_prompt_workspace_contents_and_replays(gdn, dev):
    """Captured calls follow new lengths, slots and values; the workspace's contents do not matter."""
    f = inputs([100, 30, 70], dev, 18, (1,), rows=256)
    ws = gdn.PromptWorkspace(256, 3, dev)
    ws.buf.fill_(0xFF)
    out = torch.zeros((256, HV * D), dtype=torch.bfloat16, device=dev)
    call(gdn, f, ws, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(gdn, f, ws, out=out)
    for step, lens in enumerate([[100, 30, 70], [1, 200, 3], [0, 256, 0], [64, 64, 128]]):
        n = inputs(lens, dev, 30 + step, (step % 3,), rows=256)
        for k, t in n.items():
            f[k].copy_(t)
        out.zero_()
        ws.buf.fill_(0x7F)
        g.replay()
        torch.cuda.synchronize()
        eager = call(gdn, n, out=torch.zeros_like(out))
        assert torch.equal(out, eager) and torch.equal(f["h0"], n["h0"]) and torch.equal(f["conv_state"], n["conv_state"])


def test_prompt_bits_do_not_depend_on_the_batch(gdn, dev):
    """A request's outputs and state are the same bits alone and among others."""
    f = inputs([70, 150, 9], dev, 19, (1,))
    solo = {k: v.clone() for k, v in f.items()}
    out = call(gdn, f)
    for r in range(3):
        lo, hi = int(f["qsl"][r]), int(f["qsl"][r + 1])
        p = dict(solo, **{k: solo[k][lo:hi].contiguous() for k in ("mixed", "z", "a", "b")})
        p["qsl"] = torch.tensor([0, hi - lo], dtype=torch.int32, device=dev)
        p["state_idx"], p["prefix"] = solo["state_idx"][r:r + 1], solo["prefix"][r:r + 1]
        p["h0"], p["conv_state"] = solo["h0"].clone(), solo["conv_state"].clone()
        assert torch.equal(call(gdn, p), out[lo:hi])
        assert torch.equal(p["h0"][p["state_idx"]], f["h0"][p["state_idx"]])


def test_prompt_hostile_row_starts(gdn, dev):
    """Row starts outside the batch or running backwards stay inside the buffers; a good request keeps its result."""
    f = inputs([60, 60], dev, 20, rows=120)
    want = plain(f)
    good = call(gdn, {k: v.clone() for k, v in f.items()})
    f["qsl"] = torch.tensor([0, 60, 1 << 30], dtype=torch.int32, device=dev)
    out = call(gdn, f)
    assert torch.equal(out, good)
    check(out, f, want)
    f = inputs([60, 60], dev, 20, rows=120)
    f["qsl"] = torch.tensor([-(1 << 31), 60, 10], dtype=torch.int32, device=dev)
    out = call(gdn, f, out=torch.zeros_like(out))
    assert torch.equal(out[:60], good[:60]) and not bool(out[60:].any())


def codes_of(out):
    """The e4m3 codes and scales of an output's rows, by head (exact divisions, on the CPU)."""
    y = out.float().view(-1, HV, D).cpu()
    m = y.abs().amax(-1)
    inv = torch.where(m > 0, torch.full_like(m, 448) / m, torch.zeros_like(m))
    return (y * inv[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), m / 448


# from four requests on, batches of even lengths go by whole heads, a long request among short ones by columns
@pytest.mark.parametrize("lens", [[100] * 4, [65, 64, 66, 80, 9], [9] * 6, [63, 129, 128, 127, 64, 1, 0, 8, 192, 200], [700, 1, 9, 20, 3, 64],
                                  [17] * 300])
@pytest.mark.parametrize("size", [1.0, 3e4])
def test_prompt_four_requests_and_more(gdn, dev, lens, size):
    from bundles_amd.qwen36_layer.glue import linear_rows
    n, B = sum(lens), len(lens)
    print(f"prompt of {B} requests {lens[:10]} size={size}", flush=True)
    f = inputs(lens, dev, 50 + n + B, tuple(range(0, B, 3)), rows=n + 5, pad=16)
    f["mixed"][:, 2 * HK * D:] = (f["mixed"][:, 2 * HK * D:].float() * size).to(torch.bfloat16)
    f["mixed"][n:], f["z"][n:], f["a"][n:], f["b"][n:] = (float("nan") for _ in range(4))  # rows of no request
    f["state_idx"][1] = B + 3  # padded
    out = torch.full((n + 5, HV * D), 7.0, dtype=torch.bfloat16, device=dev)
    oq = linear_rows(n + 5, 4096, dev)
    want = plain(f, out)
    call(gdn, f, out=out, oq=oq)
    check(out, f, want)
    assert bool((out[n:] == 7.0).all())
    codes, scales = codes_of(out[:n])
    assert torch.equal(oq.codes.view(torch.uint8).view(-1, HV, D)[:n].cpu(), codes)
    assert torch.equal(oq.scales.view(-1, HV)[:n].cpu(), scales)


def test_prompt_replays_from_one_rule_to_the_other(gdn, dev):
    """One captured call whose lengths change between batches that go by heads and by columns."""
    f = inputs([60] * 5, dev, 61, (1,), rows=320)
    ws = gdn.PromptWorkspace(320, 5, dev)
    out = torch.zeros((320, HV * D), dtype=torch.bfloat16, device=dev)
    call(gdn, f, ws, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(gdn, f, ws, out=out)
    for step, lens in enumerate([[60] * 5, [300, 1, 1, 1, 9], [64] * 5, [0, 0, 320, 0, 0], [1] * 5, [8, 9, 100, 70, 65]]):
        n = inputs(lens, dev, 70 + step, (step % 5,), rows=320)
        for k, t in n.items():
            f[k].copy_(t)
        out.zero_()
        ws.buf.fill_(0x7F)
        g.replay()
        torch.cuda.synchronize()
        eager = call(gdn, n, out=torch.zeros_like(out))
        assert torch.equal(out, eager) and torch.equal(f["h0"], n["h0"]) and torch.equal(f["conv_state"], n["conv_state"])


def test_prompt_two_streams(gdn, dev):
    """Two calls at once, on streams and workspaces of their own, beside each other's results."""
    fs = [inputs(lens, dev, 80 + i, (0,)) for i, lens in enumerate(([900, 30], [70] * 8))]
    alone = [{k: v.clone() for k, v in f.items()} for f in fs]
    wants = [call(gdn, f) for f in alone]
    spaces = [gdn.PromptWorkspace(f["mixed"].shape[0], len(f["state_idx"]), dev) for f in fs]
    outs = [torch.empty_like(w) for w in wants]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in fs]
    for f, ws, o, s in zip(fs, spaces, outs, streams):
        call(gdn, f, ws, out=o, stream=s)
    torch.cuda.synchronize()
    for f, a, o, w in zip(fs, alone, outs, wants):
        assert torch.equal(o, w) and torch.equal(f["h0"], a["h0"]) and torch.equal(f["conv_state"], a["conv_state"])
