"""The ring's commit (q36_gdn_ring_commit) against the recurrence in 64 bits, entry by entry.

Tolerance of the folded checkpoint: fp32 throughout; the fold adds up to 16 products (16 roundings of half a step, 2^-24, of
running values no larger than the sum of magnitudes), the decays are exponentials of sums of up to 16 gates (each sum
within 16 half steps of its magnitude, which is |G|; weights e^G |G| <= 1/e of the term), and the exponential adds 2 half
steps: together within 40 half steps of sum |terms|, taken as 40 * 2^-24 of the row's sum of magnitudes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HK, HV, D, QKV, RING = 16, 32, 128, 8192, 16


@pytest.fixture(scope="module")
def gdn():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import gdn_fused
    return gdn_fused


def pools(B, T, dev, seed, wp=None, idx=torch.int64, pad=0):
    from bundles_amd import synth
    f = synth.gdn_ring_inputs(B, T, dev, seed=seed, wp=wp)
    g = torch.Generator().manual_seed(seed)
    f["window"] = torch.randn(f["window"].shape, generator=g).to(torch.bfloat16).to(dev)
    if pad:  # slots further apart than they are long
        for k in ("conv_state", "window", "d_ring", "dlo_ring", "k_ring", "klo_ring", "g_ring"):
            t = f[k]
            n = t[0].numel()
            wide = torch.zeros((t.shape[0], n + pad), dtype=t.dtype, device=dev)
            view = torch.as_strided(wide, t.shape, (n + pad,) + t[0].contiguous().stride())
            view.copy_(t)
            f[k] = view
    for k in ("state_idx", "replay_idx", "win_idx"):
        f[k] = f[k].to(idx)
    f["accepted"] = torch.randint(1, T + 1, (B,), generator=g).to(idx).to(dev)
    return f


NAMES = ("conv_state", "window", "h0", "d_ring", "dlo_ring", "k_ring", "klo_ring", "g_ring", "state_idx", "replay_idx",
         "win_idx", "write_pos", "cache_base", "accepted")


def commit(gdn, f, T, **kw):
    gdn.gdn_ring_commit(*(f[n] for n in NAMES), T=T, **kw)


def plain(f, T, room=None, advance=True):
    room = T if room is None else room
    o = {k: f[k].cpu().clone() for k in NAMES}
    h0, big = o["h0"].double(), o["h0"].double().abs()
    for r in range(len(o["accepted"])):
        si, ri, wi, acc = (int(o[k][r]) for k in ("state_idx", "replay_idx", "win_idx", "accepted"))
        if not (0 <= si < h0.shape[0] and 0 <= ri < o["d_ring"].shape[0] and 0 <= wi < o["window"].shape[0]) or acc < 1:
            continue
        acc = min(acc, T)
        o["conv_state"][si] = o["window"][wi, :, acc - 1:acc + 2]
        n, base = min(min(max(int(o["write_pos"][ri]), 0), RING) + acc, RING), int(o["cache_base"][ri]) % RING
        fold = n + room > RING
        if fold:
            for c in range(n):
                p = (base + c) % RING
                e = o["g_ring"][ri, :, p].double().exp()[:, None, None]
                d = o["d_ring"][ri, :, p].double() + o["dlo_ring"][ri, :, p].double()
                k = (o["k_ring"][ri, :, p].double() + o["klo_ring"][ri, :, p].double()).repeat_interleave(2, 0)
                t = d[:, :, None] * k[:, None, :]
                h0[si], big[si] = h0[si] * e + t, big[si] * e + t.abs()
        if advance:
            o["write_pos"][ri] = 0 if fold else n
            if fold:
                o["cache_base"][ri] = (base + n) % RING
    o["h0"], o["bound"] = h0, 40 * 2.0 ** -24 * big
    return o


def check(f, want):
    for k in NAMES:
        got = f[k].cpu()
        if k == "h0":
            assert bool(((got.double() - want["h0"]).abs() <= want["bound"]).all())
        else:
            assert torch.equal(got, want[k]), k


@pytest.mark.parametrize("T", range(1, 9))
def test_commit_windows(gdn, dev, T):
    print(f"commit T={T}", flush=True)
    f = pools(9, T, dev, 50 + T)
    want = plain(f, T)
    commit(gdn, f, T)
    check(f, want)


@pytest.mark.parametrize("room,advance,wp", [(0, True, 3), (16, True, 0), (4, False, 12), (1, True, 16), (8, True, 15)])
def test_commit_room_and_cursors(gdn, dev, room, advance, wp):
    f = pools(4, 4, dev, 7, wp=wp)
    want = plain(f, 4, room, advance)
    commit(gdn, f, 4, room=room, advance=advance)
    check(f, want)


def test_commit_int32_indices_strided_pools_and_odd_cursors(gdn, dev):
    """Cursors outside the ring, which count as the nearest inside (write_pos) and modulo 16 (cache_base)."""
    f = pools(6, 5, dev, 9, idx=torch.int32, pad=24)
    f["write_pos"][f["replay_idx"][0].long()] = -3
    f["write_pos"][f["replay_idx"][1].long()] = 99
    f["cache_base"][f["replay_idx"][2].long()] = 37
    f["write_pos"][f["replay_idx"][3].long()] = 12
    f["cache_base"][f["replay_idx"][3].long()] = -1
    want = plain(f, 5)
    commit(gdn, f, 5)
    check(f, want)


def test_commit_padded_requests(gdn, dev):
    f = pools(7, 4, dev, 10, wp=12)
    f["state_idx"][0] = -1
    f["replay_idx"][1] = 1 << 40
    f["win_idx"][2] = f["window"].shape[0]
    f["accepted"][3] = 0
    f["accepted"][4] = -7
    f["accepted"][5] = 100
    want = plain(f, 4)
    commit(gdn, f, 4)
    check(f, want)


def test_commit_extreme_gates(gdn, dev):
    """Decays that leave nothing, and none at all; entries behind the history hold NaN."""
    f = pools(5, 4, dev, 12, wp=9)
    f["g_ring"][0] = -1000.0
    f["g_ring"][1] = 0.0
    for b in range(5):
        ri = int(f["replay_idx"][b])
        n = 9 + int(f["accepted"][b])
        for c in range(n, RING):
            p = (int(f["cache_base"][ri]) + c) % RING
            for k in ("d_ring", "dlo_ring", "k_ring", "klo_ring", "g_ring"):
                f[k][ri, :, p] = float("nan")
    want = plain(f, 4, 16)
    commit(gdn, f, 4, room=16)
    for k in ("conv_state", "write_pos", "cache_base"):
        assert torch.equal(f[k].cpu(), want[k])
    assert bool(((f["h0"].cpu().double() - want["h0"]).abs() <= want["bound"]).all())


def test_commit_window_view_and_graph(gdn, dev):
    T = 4
    f = pools(5, T, dev, 14, wp=5)
    win = f["window"]
    g = torch.cuda.CUDAGraph()
    before = {k: f[k].clone() for k in NAMES}
    view = torch.as_strided(win, (win.shape[0], T, QKV, 3), (win.stride(0), 1, T + 2, 1))

    def call():
        gdn.gdn_ring_commit(f["conv_state"], view, *(f[n] for n in NAMES[2:]), T=T)
    call()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        call()
    for step in range(4):
        want = plain(f, T)
        g.replay()
        torch.cuda.synchronize()
        check(f, want)
        f["accepted"].copy_(torch.randint(1, T + 1, (5,), generator=torch.Generator().manual_seed(step)))
    assert not torch.equal(before["write_pos"], f["write_pos"])
