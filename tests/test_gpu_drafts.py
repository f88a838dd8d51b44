"""Verification of drafts (q36_verify_drafts) against a sequential statement of it in 64 bits, token for token."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_lmhead8 import lmhead8
    return lmhead8


def plain(logits, drafts, uniforms, temperature, probs):
    """logits fp64 [B, T, V]; the definition, one request after another."""
    B, T, V = logits.shape
    tokens, counts = np.full((B, T), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        heat = 1.0 if temperature is None else temperature[b]
        j = 0
        while True:
            x = np.where(np.isnan(logits[b, j]), -np.inf, logits[b, j])
            m = x.max()
            if m == -np.inf:
                counts[b] = j
                break
            if heat > 0:
                with np.errstate(invalid="ignore"):
                    p = np.where(x == m, 1.0, np.nan_to_num(np.exp((x - m) / heat), nan=0.0))
                p = p / p.sum()
            else:
                p = (np.arange(V) == int(np.argmax(x))).astype(float)
            d = drafts[b, j] if j < T - 1 else -1
            left = p
            if 0 <= d < V:
                q = np.zeros(V) if probs is None else probs[b, j].astype(float)
                if probs is None:
                    q[d] = 1.0
                if float(uniforms[b, j]) * q[d] < p[d]:
                    tokens[b, j] = d
                    j += 1
                    continue
                left = np.maximum(p - q, 0)
                if left.sum() <= 0:
                    left = p
            run = np.cumsum(left)
            over = np.nonzero((run > float(uniforms[b, T - 1]) * run[-1]) & (left > 0))[0]
            tokens[b, j] = over[0] if len(over) else np.nonzero(left > 0)[0][-1]
            counts[b] = j + 1
            break
    return tokens, counts


def compare(lm, logits, drafts, uniforms, temperature=None, probs=None, ws=None):
    B, T = uniforms.shape
    V = logits.shape[1]
    ws = ws or lm.VerifyWorkspace(B, T, V, logits.device)
    ws.buf.fill_(0xA5)
    tokens, counts = lm.verify_drafts(logits, drafts if T > 1 else None, uniforms, ws, temperature=temperature,
                                      draft_probs=probs)
    torch.cuda.synchronize()
    cpu = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    want = plain(logits.cpu().double().view(B, T, V).numpy(), cpu(drafts), cpu(uniforms), cpu(temperature), cpu(probs))
    assert np.array_equal(counts.cpu().numpy(), want[1])
    assert np.array_equal(tokens.cpu().numpy(), want[0])
    return counts.cpu().numpy()


def inputs(B, T, V, dev, seed, dtype=torch.bfloat16, probs=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((B * T, V), generator=g) * 2 + 5 * (torch.rand((B * T, V), generator=g) < 0.01)).to(torch.bfloat16)
    near = x.float().view(B, T, V)[:, :-1] + 0.5 * torch.randn((B, T - 1, V), generator=g)
    q = torch.softmax(near, -1) if probs else None
    if T == 1:
        drafts = torch.zeros((B, 0), dtype=torch.int32)
    elif probs:
        drafts = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, T - 1).to(torch.int32)
    else:
        drafts = near.argmax(-1).to(torch.int32)
    u = torch.rand((B, T), generator=g)
    heat = 0.3 + torch.rand(B, generator=g)
    return x.to(dtype).to(dev), drafts.to(dev), u.to(dev), heat.to(dev), None if q is None else q.to(dev)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 1, 4097), (5, 4, 1000), (2, 8, 8191), (7, 5, 4096), (2, 3, 65537), (33, 2, 16)])
def test_drafts_sizes(lm, dev, B, T, V, probs, dtype):
    print(f"drafts B={B} T={T} V={V} probs={probs} {dtype}", flush=True)
    x, d, u, heat, q = inputs(B, T, V, dev, 11 * B + T + V, dtype, probs and T > 1)
    compare(lm, x, d, u, heat, q)
    compare(lm, x, d, u, None, q)


def test_drafts_full_vocabulary(lm, dev):
    x, d, u, heat, q = inputs(6, 5, 151936, dev, 3, probs=True)
    heat[1] = 0.0
    heat[4] = float("nan")  # greedy
    n = compare(lm, x, d, u, heat, q)
    assert n.min() < n.max()


def test_drafts_greedy_takes_the_first_largest(lm, dev):
    """Ties go to the lowest index, in one segment and across segments."""
    V = 9000
    x = torch.zeros((4 * 3, V), dtype=torch.bfloat16)
    x[:, [17, 5000, 8999]] = 3.0
    x[3:6, 17] = 0.0
    d = torch.tensor([[17, 17], [5000, 5000], [17, 5000], [8999, 17]], dtype=torch.int32)
    u = torch.full((4, 3), 0.999)
    n = compare(lm, x.to(dev), d.to(dev), u.to(dev), torch.zeros(4, device=dev))
    assert n.tolist() == [3, 3, 2, 1]


def test_drafts_masked_rows_infinities_nan(lm, dev):
    """Rows of minus infinity alone, NaN logits, infinite logits, masked vocabularies, drafts that are none."""
    B, T, V = 8, 3, 5003
    x, d, u, heat, _ = inputs(B, T, V, dev, 21)
    x, d = x.view(B, T, V), d
    x[0, 0] = float("-inf")                        # nothing from the start
    x[1, 1] = float("nan")
    d[1, 0] = x[1, 0].float().argmax().int()
    u[1, 0] = 0.0                                  # the first draft stands, then nothing is left
    x[2, :, 100:] = float("-inf")
    x[3, 0, ::2] = float("nan")
    x[4, 0, [7, 4999]] = float("inf")              # share the row
    d[5, 0] = -1
    d[6, 0] = V
    x[7, 0] = torch.finfo(torch.bfloat16).min      # a mask of the lowest value: even
    x[7, 0, 4200] = 0.0
    for probs in (None, torch.softmax(torch.randn((B, T - 1, V), device=dev), -1)):
        n = compare(lm, x.view(B * T, V), d, u, heat, probs)
        assert n[0] == 0 and n[1] in (1,), n


def test_drafts_ends_of_the_random_range(lm, dev):
    x, d, u, heat, q = inputs(4, 2, 4500, dev, 5, probs=True)
    for v in (0.0, 1.0 - 2.0 ** -24):
        u.fill_(v)
        compare(lm, x, d, u, heat, q)
        compare(lm, x, d, u, heat)
    q.copy_(torch.softmax(x.float().view(4, 2, -1)[:, :1], -1))  # p = q: nothing is left but rounding, or p itself
    u.fill_(1.0)
    tok, n = lm.verify_drafts(x, d, u, lm.VerifyWorkspace(4, 2, 4500, dev), draft_probs=q)
    assert ((tok >= 0).sum(1) == n).all()


def test_drafts_cold_and_hot(lm, dev):
    x, d, u, heat, _ = inputs(5, 4, 5000, dev, 6)
    heat.copy_(torch.tensor([1e-6, 1e-40, 1e30, float("inf"), -1.0]))
    h = heat.clone()
    h[1] = 1e-40
    B, T, V = 5, 4, 5000
    tokens, counts = lm.verify_drafts(x, d, u, lm.VerifyWorkspace(B, T, V, dev), temperature=h)
    want = h.cpu().double().numpy()
    want[3] = 1e30
    ref = plain(x.cpu().double().view(B, T, V).numpy(), d.cpu().numpy(), u.cpu().numpy(), want, None)
    assert np.array_equal(tokens.cpu().numpy(), ref[0]) and np.array_equal(counts.cpu().numpy(), ref[1])


def test_drafts_strided_rows_and_alignment(lm, dev):
    """Rows inside a wider buffer, 16-byte aligned and not."""
    x, d, u, heat, _ = inputs(3, 4, 4100, dev, 8)
    for pad, off in ((12, 0), (12, 8), (13, 0), (12, 1)):
        wide = torch.full((12, 4100 + pad), 100.0, dtype=torch.bfloat16, device=dev)
        rows = wide[:, off:off + 4100]
        rows.copy_(x)
        compare(lm, rows, d, u, heat)


def test_drafts_draws_follow_the_probabilities(lm, dev):
    """Evenly spaced numbers through one row: each token comes as often as its probability says, to one."""
    V, N = 37, 4096
    x = torch.randn((1, V), generator=torch.Generator().manual_seed(2)).repeat(N, 1).to(dev)
    u = ((torch.arange(N, dtype=torch.float64) + 0.5) / N).float()[:, None].to(dev)
    tok, n = lm.verify_drafts(x, None, u, lm.VerifyWorkspace(N, 1, V, dev))
    share = torch.bincount(tok[:, 0].cpu().long(), minlength=V).double()
    assert (share - torch.softmax(x[0].cpu().double(), -1) * N).abs().max() <= 1.0 + 1e-3


def test_drafts_graph_replays(lm, dev):
    x, d, u, heat, q = inputs(6, 4, 6001, dev, 13, probs=True)
    ws = lm.VerifyWorkspace(6, 4, 6001, dev)
    tok, n = torch.empty((6, 4), dtype=torch.int32, device=dev), torch.empty(6, dtype=torch.int32, device=dev)
    lm.verify_drafts(x, d, u, ws, heat, q, tok, n)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lm.verify_drafts(x, d, u, ws, heat, q, tok, n)
    for k in range(4):
        x2, d2, u2, h2, q2 = inputs(6, 4, 6001, dev, 100 + k, probs=True)
        for a, b in ((x, x2), (d, d2), (u, u2), (heat, h2), (q, q2)):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        got = tok.clone(), n.clone()
        want = lm.verify_drafts(x2, d2, u2, ws, h2, q2)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype,probs,V", [(torch.bfloat16, False, 50001), (torch.float32, True, 50008), (torch.bfloat16, True, 131071)])
def test_drafts_large_calls(lm, dev, dtype, probs, V):
    """Calls large enough that the rows' sums are fp32 and the drawn row alone is summed in fp64; some requests greedy."""
    B, T = 25200000 // (3 * V) + 1, 4
    print(f"drafts B={B} T={T} V={V} probs={probs} {dtype}", flush=True)
    x, d, u, heat, q = inputs(B, T, V, dev, V, dtype, probs)
    heat[::5] = 0.0
    n = compare(lm, x, d, u, heat, q)
    assert n.min() < n.max()


def test_drafts_numbers_at_the_border(lm, dev):
    """Numbers within an fp32 step of the drafts' probabilities, on either side, in a call whose sums are fp32: the tests
    come out as with sums in 64 bits."""
    B, T, V = 130, 4, 65544
    x, d, u, heat, _ = inputs(B, T, V, dev, 77)
    y = x.cpu().double().view(B, T, V) / heat.cpu().double()[:, None, None]
    p = torch.softmax(y, -1)[:, :-1].gather(-1, d.cpu().long()[..., None])[..., 0]
    near = p.float()
    near[::3] = torch.nextafter(near[::3], torch.zeros(()))
    near[1::3] = torch.nextafter(near[1::3], torch.ones(()))
    assert float(((near.double() - p).abs() / p).max()) < 2.0 ** -22
    u[:, :-1] = near.to(dev)
    n = compare(lm, x, d, u, heat)
    assert {1, 2} <= set(n.tolist())


def test_drafts_large_graph_and_two_streams(lm, dev):
    """The large form replayed with new values, and beside another call on a stream and workspace of its own."""
    B, T, V = 130, 4, 65544
    x, d, u, heat, _ = inputs(B, T, V, dev, 78)
    ws = lm.VerifyWorkspace(B, T, V, dev)
    tok, n = torch.empty((B, T), dtype=torch.int32, device=dev), torch.empty(B, dtype=torch.int32, device=dev)
    lm.verify_drafts(x, d, u, ws, heat, None, tok, n)
    first = tok.clone(), n.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lm.verify_drafts(x, d, u, ws, heat, None, tok, n)
    seen = []
    for k in range(3):
        u.copy_(torch.rand((B, T), generator=torch.Generator().manual_seed(k)))
        ws.buf.fill_(0xFF)
        g.replay()
        torch.cuda.synchronize()
        seen.append((u.clone(), tok.clone(), n.clone()))
        want = lm.verify_drafts(x, d, u, lm.VerifyWorkspace(B, T, V, dev), heat)
        assert torch.equal(tok, want[0]) and torch.equal(n, want[1])
    assert not torch.equal(seen[0][1], first[0])
    spaces, streams, got = [lm.VerifyWorkspace(B, T, V, dev) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(2):
        got.append(lm.verify_drafts(x, d, seen[i][0], spaces[i], heat, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i][0], seen[i][1]) and torch.equal(got[i][1], seen[i][2])
