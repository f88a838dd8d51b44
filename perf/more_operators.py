"""The operators around a request's recurrent state and its drafts, with their plain forms: the prompt of a recurrent
layer, the verification of drafted tokens, and the commit of what was accepted to the recurrent state.

A case is a dict of plain values; its "kind" names the operator:
  prompt  gdn_fused.gdn_prompt: causal conv, gates, the gated delta rule over any number of new tokens a request, gated
          norm; conv state and recurrent state carried in the pools
  verify  lmhead8.verify_drafts: drafts accepted or refused against the target's probabilities, the next token drawn
  commit  gdn_fused.gdn_ring_commit: conv state, ring cursor and checkpoint moved to the accepted position
The recurrent layer's widths are fixed: 16 key heads and 32 value heads of 128, a conv of 4 taps over 8192 channels.

Lengths follow from the case alone, values from the seed: request b's length lies between the case's bounds, spread
evenly over the logarithm, in an order that mixes long and short ones.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HK, HV, D, QKV, RING = 16, 32, 128, 8192, 16
BF, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
EPS, SCALE, C = 1e-6, 128 ** -0.5, 64


def listed():
    return [
        # five decoding requests, one new token each: latency, and 2 MB of state in and out a request
        dict(name="prompt_5x1", kind="prompt", B=5, new_min=1, new_max=1, fresh_every=0),
        # one short prompt from an empty state
        dict(name="prompt_1x517", kind="prompt", B=1, new_min=517, new_max=517, fresh_every=1),
        # a mixed serving step: decoding requests beside prompts, every third of them new
        dict(name="prompt_mixed_24", kind="prompt", B=24, new_min=1, new_max=900, fresh_every=3),
        # the next piece of one long prompt: nothing but the sequence itself to spread over the chip
        dict(name="prompt_1x8192", kind="prompt", B=1, new_min=8192, new_max=8192, fresh_every=0),
        # the largest batch: 16 new prompts of a thousand tokens
        dict(name="prompt_16x1000", kind="prompt", B=16, new_min=1000, new_max=1000, fresh_every=1),
        # sampling one token of one request: no draft
        dict(name="verify_1x1", kind="verify", B=1, T=1, V=151936, logits="bf16", probs=False, greedy_every=0),
        # the verify window of the reference, greedy and sampled requests mixed, greedy drafts
        dict(name="verify_32x4", kind="verify", B=32, T=4, V=151936, logits="f32", probs=False, greedy_every=4),
        # drafts that were sampled from a draft model, whose probabilities come along
        dict(name="verify_64x5", kind="verify", B=64, T=5, V=151936, logits="bf16", probs=True, greedy_every=0),
        # the lm_head's largest batch of rows, a small vocabulary of an odd size beside it in the draws
        dict(name="verify_256x8", kind="verify", B=256, T=8, V=151936, logits="bf16", probs=False, greedy_every=0),
        # three requests; the cursors move on with the call
        dict(name="commit_3x4", kind="commit", B=3, T=4, advance=True),
        # a full verify batch of one layer, as the layers before the last commit it
        dict(name="commit_64x4", kind="commit", B=64, T=4, advance=False),
        # the largest batch, the longest window
        dict(name="commit_256x8", kind="commit", B=256, T=8, advance=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "verify", "commit"])
    if kind == "prompt":
        # 1 .. 64 requests of 1 .. 8191 new tokens, none, some or all of them new
        while True:
            B, new = _log_int(rng, 1, 64), _log_int(rng, 1, 8191)
            if B * new <= 16000:
                break
        return dict(kind=kind, B=B, new_min=rng.randint(1, new), new_max=new, fresh_every=rng.choice([0, 1, 2, 3]))
    if kind == "verify":
        # 1 .. 256 requests, 0 .. 7 drafts, vocabularies of 1000 .. 151936, odd ones among them
        while True:
            B, T, V = _log_int(rng, 1, 256), rng.randint(1, 8), _log_int(rng, 1000, 151936)
            if B * T * V <= 2048 * 151936 // 4:
                break
        return dict(kind=kind, B=B, T=T, V=V, logits=rng.choice(["bf16", "f32"]), probs=T > 1 and rng.random() < 0.4,
                    greedy_every=rng.choice([0, 0, 1, 3]))
    # 1 .. 250 requests, every window
    return dict(kind=kind, B=_log_int(rng, 1, 250), T=rng.randint(1, 8), advance=rng.random() < 0.5)


# ---- what follows from the case alone ---------------------------------------------------------------------
def _spread(B, lo, hi):
    """B lengths from lo to hi, evenly over the logarithm, the longest among them."""
    if B == 1:
        return [hi]
    order = sorted(range(B), key=lambda b: (b * 0.6180339887498949) % 1.0)
    out = [0] * B
    for k, b in enumerate(order):
        u = k / (B - 1)
        out[b] = int(round(lo ** (1 - u) * hi ** u))
    return out


def _lengths(c):
    return _spread(c["B"], c["new_min"], c["new_max"])


def _fresh(c):
    return [c["fresh_every"] > 0 and b % c["fresh_every"] == 0 for b in range(c["B"])]


def _cursors(c):
    """Committed entries before the window, and accepted tokens, of each request."""
    return [(5 * b + 3) % (RING - c["T"] + 1) for b in range(c["B"])], [1 + (3 * b) % c["T"] for b in range(c["B"])]


# ---- inputs ---------------------------------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + salt)
    return g


def _randn(shape, g, std=1.0, dtype=BF):
    return (torch.randn(shape, generator=g, device=DEV, dtype=F32) * std).to(dtype)


def _ints(v, dtype=I32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def _pick(n, B, g):
    return torch.randperm(n, generator=g, device=DEV)[:B].contiguous()


def _gates(g):
    """A_log and dt_bias of the gate: decay rates from 1 to 16, time steps from 1e-3 to 1e-1."""
    dt = torch.exp(torch.rand(HV, generator=g, device=DEV) * math.log(100.0) + math.log(1e-3))
    return torch.log(1 + 15 * torch.rand(HV, generator=g, device=DEV)), dt + torch.log(-torch.expm1(-dt))


def prepare(case, seed):
    c, kind, B = case, case["kind"], case["B"]
    if kind == "prompt":
        g, n = _gen(seed, 1), _lengths(c)
        T, slots = sum(n), B + 2
        A_log, dt_bias = _gates(g)
        fresh = _fresh(c)
        return dict(kind=kind, c=c, n=n, mixed=_randn((T, QKV), g), z=_randn((T, HV * D), g), a=_randn((T, HV), g),
                    b=_randn((T, HV), g), conv_state=_randn((slots, QKV, 3), g),
                    conv_w=(torch.rand((QKV, 4), generator=g, device=DEV) - 0.5).to(BF), A_log=A_log, dt_bias=dt_bias,
                    h0=torch.randn((slots, HV, D, D), generator=g, device=DEV) * 0.1, norm_w=_randn((D,), g, 0.1) + 1.0,
                    qsl=_ints([sum(n[:b]) for b in range(B + 1)]), slot=_pick(slots, B, g),
                    prefix=_ints([0 if f else 77 + b for b, f in enumerate(fresh)]))
    if kind == "verify":
        g, T, V = _gen(seed, 2), c["T"], c["V"]
        # logits with a heavy head, as a trained model's, rounded to bf16 as the lm_head leaves them
        x = torch.randn((B * T, V), generator=g, device=DEV)
        x = (x * 2.0 + 6.0 * (torch.rand((B * T, V), generator=g, device=DEV) < 3e-4)).to(BF)
        if T > 1:
            noise = torch.randn((B, T - 1, V), generator=g, device=DEV)
            near = x.view(B, T, V)[:, :-1].to(F32) + 0.7 * noise
            del noise
        probs = None
        if T > 1 and c["probs"]:
            probs = torch.softmax(near, dim=-1)
            drafts = torch.multinomial(probs.view(-1, V), 1, generator=g).view(B, T - 1).to(I32)
        else:
            drafts = near.argmax(-1).to(I32) if T > 1 else torch.zeros((B, 0), dtype=I32, device=DEV)
        greedy = [c["greedy_every"] > 0 and b % c["greedy_every"] == 0 for b in range(B)]
        temperature = 0.5 + torch.rand(B, generator=g, device=DEV)
        temperature = torch.where(torch.tensor(greedy, device=DEV), torch.zeros_like(temperature), temperature)
        return dict(kind=kind, c=c, logits=x.to(F32) if c["logits"] == "f32" else x, drafts=drafts.contiguous(), probs=probs,
                    uniforms=torch.rand((B, T), generator=g, device=DEV), temperature=temperature)
    g, T = _gen(seed, 3), c["T"]
    slots, rslots, wslots = B + 3, B + 2, B + 1
    wp, acc = _cursors(c)
    state_idx, replay_idx, win_idx = _pick(slots, B, g), _pick(rslots, B, g), _pick(wslots, B, g)
    write_pos = torch.zeros(rslots, dtype=I32, device=DEV)
    write_pos[replay_idx] = _ints(wp)
    d = torch.randn((rslots, HV, RING, D), generator=g, device=DEV) * 0.3
    k = torch.randn((rslots, HK, RING, D), generator=g, device=DEV)
    k = k / k.norm(dim=-1, keepdim=True)
    A_log, dt_bias = _gates(g)
    gate = torch.randn((rslots, HV, RING), generator=g, device=DEV) + dt_bias[None, :, None]
    return dict(kind=kind, c=c, conv_state=_randn((slots, QKV, 3), g), window=_randn((wslots, QKV, T + 2), g),
                h0=torch.randn((slots, HV, D, D), generator=g, device=DEV) * 0.1,
                d=d.to(BF), dlo=(d - d.to(BF).to(F32)).to(BF), k=k.to(BF), klo=(k - k.to(BF).to(F32)).to(BF),
                g=-torch.exp(A_log)[None, :, None] * torch.nn.functional.softplus(gate),
                state_idx=state_idx, replay_idx=replay_idx, win_idx=win_idx, write_pos=write_pos,
                cache_base=torch.randint(0, RING, (rslots,), generator=g, device=DEV, dtype=I32), accepted=_ints(acc))


# ---- the prompt -------------------------------------------------------------------------------------------------
def _prompt_plain(s):
    n, B, N = s["n"], len(s["n"]), max(s["n"])
    NC = -(-N // C)
    qsl, slot, old = s["qsl"].long(), s["slot"], (s["prefix"] > 0)
    t = torch.arange(NC * C, device=DEV)
    here = t[None] < (qsl[1:] - qsl[:-1])[:, None]                                  # [B, N']
    row = torch.where(here, qsl[:-1, None] + t, torch.zeros_like(t))
    x = torch.where(here[..., None], s["mixed"][row], torch.zeros((), dtype=BF, device=DEV))
    before = torch.where(old[:, None, None], s["conv_state"][slot], torch.zeros((), dtype=BF, device=DEV))
    ext = torch.cat([before.transpose(1, 2), x], dim=1).to(F32)                   # [B, 3 + N', 8192]
    w = s["conv_w"].to(F32)
    y = ext[:, :-3] * w[:, 0] + ext[:, 1:-2] * w[:, 1] + ext[:, 2:-1] * w[:, 2] + ext[:, 3:] * w[:, 3]
    y = y * torch.sigmoid(y)
    ends = torch.arange(3, device=DEV) + (qsl[1:] - qsl[:-1])[:, None]
    s["conv_state"][slot] = ext[torch.arange(B, device=DEV)[:, None], ends].to(BF).transpose(1, 2)
    q, k, v = (p.reshape(B, NC, C, h, D).transpose(2, 3) for p, h in
               zip(y.split([HK * D, HK * D, HV * D], dim=-1), (HK, HK, HV)))        # [B, NC, heads, C, D]
    del y, ext, x
    q = (q * torch.rsqrt(q.square().sum(-1, keepdim=True) + 1e-6) * SCALE).repeat_interleave(HV // HK, dim=2)
    k = (k * torch.rsqrt(k.square().sum(-1, keepdim=True) + 1e-6)).repeat_interleave(HV // HK, dim=2)
    gate = s["a"].to(F32) + s["dt_bias"]
    gate = -torch.exp(s["A_log"]) * torch.where(gate > 20, gate, torch.log1p(torch.exp(gate.clamp(max=20))))
    gate, beta = (torch.where(here[..., None], p[row], torch.zeros((), device=DEV)).view(B, NC, C, HV).transpose(2, 3)
                  for p in (gate, torch.sigmoid(s["b"].to(F32))))                   # [B, NC, 32, C]
    run = torch.cumsum(gate.to(F64), -1)                                            # a long sum
    fade = torch.exp((run[..., :, None] - run[..., None, :]).tril()).to(F32).tril()  # e^(b_i - b_j), j <= i
    run, rest = torch.exp(run).to(F32), torch.exp(run[..., -1:] - run).to(F32)
    kt = k.transpose(-1, -2).contiguous()
    A = (torch.matmul(k, kt) * fade * beta[..., None]).tril(-1) + torch.eye(C, device=DEV)
    P = torch.matmul(q, kt) * fade
    S = torch.where(old[:, None, None, None], s["h0"][slot], torch.zeros((), device=DEV)).transpose(-1, -2).contiguous()
    o = torch.empty((B, NC, HV, C, D), device=DEV)
    for i in range(NC):
        X = beta[:, i, :, :, None] * (v[:, i] - run[:, i, :, :, None] * torch.matmul(k[:, i], S))
        U = torch.linalg.solve_triangular(A[:, i], X, upper=False, unitriangular=True)
        o[:, i] = run[:, i, :, :, None] * torch.matmul(q[:, i], S) + torch.matmul(P[:, i], U)
        S = run[:, i, :, -1, None, None] * S + torch.matmul(kt[:, i], rest[:, i, :, :, None] * U)
    s["h0"][slot] = S.transpose(-1, -2)
    o = o.transpose(2, 3).reshape(B, NC * C, HV, D)[here]
    z = s["z"].view(-1, HV, D).to(F32)
    out = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["norm_w"].to(F32) * (z * torch.sigmoid(z))
    return [out.view(-1, HV * D).to(BF), s["conv_state"], s["h0"]]


def _prompt_own(s):
    from bundles_amd.qwen36_layer import gdn_fused
    if "ws" not in s:
        s["ws"] = gdn_fused.PromptWorkspace(s["mixed"].shape[0], len(s["n"]), DEV)
    out = gdn_fused.gdn_prompt(s["mixed"], s["z"], s["a"], s["b"], s["conv_state"], s["conv_w"], s["A_log"], s["dt_bias"],
                               s["h0"], s["qsl"], s["slot"], s["norm_w"], s["ws"], EPS, SCALE, prefix=s["prefix"])
    return [out, s["conv_state"], s["h0"]]


# ---- the verification of drafts -----------------------------------------------------------------------------------
def _verify_plain(s):
    c = s["c"]
    B, T, V = c["B"], c["T"], c["V"]
    x = s["logits"].view(B, T, V).to(F64)  # running sums over the vocabulary, and tests beside a border
    top, best = x.max(-1)
    best = torch.where(x == top[..., None], torch.arange(V, device=DEV), V).amin(-1)
    heat = s["temperature"].to(F64)[:, None]
    greedy = heat <= 0
    x = x.sub_(top[..., None]).div_(torch.where(greedy, torch.ones_like(heat), heat)[..., None]).exp_()
    norm = x.sum(-1)
    b = torch.arange(B, device=DEV)
    tok, u = s["drafts"].long(), s["uniforms"].to(F64)
    p = x[:, :-1].gather(-1, tok[..., None])[..., 0] / norm[:, :-1]
    p = torch.where(greedy, (best[:, :-1] == tok).to(F64), p)
    q = torch.ones_like(p) if s["probs"] is None else s["probs"].gather(-1, tok[..., None])[..., 0].to(F64)
    j = torch.cumprod((u[:, :-1] * q < p).to(I64), -1).sum(-1)                      # accepted drafts
    w = x[b, j] / norm[b, j][:, None]
    w = torch.where(greedy, (torch.arange(V, device=DEV) == best[b, j][:, None]).to(F64), w)
    if T > 1:
        jd = j.clamp(max=T - 2)
        less = torch.zeros_like(w).scatter_(1, tok[b, jd][:, None], 1.0) if s["probs"] is None else s["probs"][b, jd].to(F64)
        r = torch.where((j < T - 1)[:, None], (w - less).clamp(min=0), w)
        w = torch.where(r.sum(-1, keepdim=True) > 0, r, w)
    run = torch.cumsum(w, -1)
    nxt = torch.searchsorted(run, (u[:, -1] * run[:, -1])[:, None], right=True)[:, 0]
    last = torch.where(w > 0, torch.arange(V, device=DEV), 0).amax(-1)
    nxt = torch.minimum(nxt, last)
    i = torch.arange(T, device=DEV)
    tokens = torch.where(i < j[:, None], torch.cat([tok, nxt[:, None]], 1), torch.full((), -1, dtype=I64, device=DEV))
    tokens = torch.where(i == j[:, None], nxt[:, None], tokens)
    return [tokens.to(I32), (j + 1).to(I32)]


def _verify_own(s):
    from bundles_amd.qwen36_lmhead8 import lmhead8
    c = s["c"]
    if "ws" not in s:
        s["ws"] = lmhead8.VerifyWorkspace(c["B"], c["T"], c["V"], DEV)
    return list(lmhead8.verify_drafts(s["logits"], s["drafts"], s["uniforms"], s["ws"], temperature=s["temperature"],
                                      draft_probs=s["probs"]))


# ---- the commit -----------------------------------------------------------------------------------------------------
def _commit_plain(s):
    c, B = s["c"], s["c"]["B"]
    si, ri, wi, acc = s["state_idx"], s["replay_idx"], s["win_idx"], s["accepted"].long()
    b = torch.arange(B, device=DEV)
    tap = (acc - 1)[:, None, None] + torch.arange(3, device=DEV)
    s["conv_state"][si] = s["window"][wi].gather(2, tap.expand(B, QKV, 3))
    base = s["cache_base"][ri].long()
    n = s["write_pos"][ri].long() + acc
    fold = n + c["T"] > RING
    e = torch.arange(RING, device=DEV)
    at = (base[:, None] + e) % RING                                                   # physical slot of entry e
    on = (e < n[:, None])[:, None]                                                    # [B, 1, 16]
    g = s["g"][ri].gather(2, at[:, None].expand(B, HV, RING)).to(F64) * on
    run = torch.cumsum(g, -1)                                                         # [B, 32, 16]
    fade = (torch.exp(run[..., -1:] - run) * on).to(F32)
    d, k = (s[h][ri[:, None], :, at].to(F32) + s[l][ri[:, None], :, at].to(F32) for h, l in (("d", "dlo"), ("k", "klo")))
    d = torch.where(on[..., None], d.transpose(1, 2) * fade[..., None], torch.zeros((), device=DEV))  # [B, 32, 16, 128]
    k = torch.where(on[..., None], k.transpose(1, 2), torch.zeros((), device=DEV)).repeat_interleave(HV // HK, dim=1)
    old = s["h0"][si]
    new = torch.exp(run[..., -1]).to(F32)[..., None, None] * old + torch.matmul(d.transpose(-1, -2).contiguous(), k)
    s["h0"][si] = torch.where(fold[:, None, None, None], new, old)
    if c["advance"]:
        s["write_pos"][ri] = torch.where(fold, torch.zeros_like(n), n).to(I32)
        s["cache_base"][ri] = torch.where(fold, (base + n) % RING, base).to(I32)
    return [s["conv_state"], s["h0"], s["write_pos"], s["cache_base"]]


def _commit_own(s):
    from bundles_amd.qwen36_layer import gdn_fused
    gdn_fused.gdn_ring_commit(s["conv_state"], s["window"], s["h0"], s["d"], s["dlo"], s["k"], s["klo"], s["g"], s["state_idx"],
                              s["replay_idx"], s["win_idx"], s["write_pos"], s["cache_base"], s["accepted"], T=s["c"]["T"],
                              advance=s["c"]["advance"])
    return [s["conv_state"], s["h0"], s["write_pos"], s["cache_base"]]


def run(state):
    kind = state["kind"]
    if kind == "prompt":
        return _prompt_own(state) if own else _prompt_plain(state)
    if kind == "verify":
        return _verify_own(state) if own else _verify_plain(state)
    return _commit_own(state) if own else _commit_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    c, kind, B = case, case["kind"], case["B"]
    if kind == "prompt":
        T, old = sum(_lengths(c)), B - sum(_fresh(c))
        state, conv = 4 * HV * D * D, 2 * 3 * QKV
        return {"bytes": T * (2 * QKV + 4 * HV * D + 4 * HV) + (B + old) * (state + conv) + 8 * QKV + 16 * B,
                "flops": T * HV * 6 * D * D}
    if kind == "verify":
        T, V = c["T"], c["V"]
        per = 2 if c["logits"] == "bf16" else 4
        # every logit once (a row behind a refusal is known as such only once the rows before are summed), and one row of
        # draft probabilities a request
        return {"bytes": B * (T * V * per + (4 * V if c["probs"] else 0) + 12 * T), "flops": B * T * V * 4}
    T = c["T"]
    wp, acc = _cursors(c)
    folds = [w + a for w, a in zip(wp, acc) if w + a + T > RING]
    ring = sum(n * (2 * 2 * HV * D + 2 * 2 * HK * D + 4 * HV) for n in folds)
    return {"bytes": B * (2 * 2 * 3 * QKV + 20) + len(folds) * 2 * 4 * HV * D * D + ring, "flops": sum(folds) * HV * 2 * D * D}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "verify":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "commit":
        conv, h0 = s["conv_state"].double(), s["h0"].double()
        wp, acc = _cursors(case)
        for b in range(case["B"]):
            si, ri, wi = int(s["state_idx"][b]), int(s["replay_idx"][b]), int(s["win_idx"][b])
            conv[si] = s["window"][wi, :, acc[b] - 1:acc[b] + 2].double()
            n = wp[b] + acc[b]
            if n + case["T"] <= RING:
                continue
            for e in range(n):
                p = (int(s["cache_base"][ri]) + e) % RING
                d = s["d"][ri, :, p].double() + s["dlo"][ri, :, p].double()
                k = (s["k"][ri, :, p].double() + s["klo"][ri, :, p].double()).repeat_interleave(HV // HK, 0)
                h0[si] = h0[si] * s["g"][ri, :, p].double().exp()[:, None, None] + d[:, :, None] * k[:, None, :]
        return [conv, h0, None, None]
    n, B = s["n"], case["B"]
    if B * max(n) * HV * D * D * 8 * 6 / 3e12 + max(n) * 8e-5 > 15:
        return None
    N, T = max(n), sum(n)
    conv, h0, slot = s["conv_state"].double(), s["h0"].double(), s["slot"]
    fresh = torch.tensor(_fresh(case), device=DEV)
    S = h0[slot].masked_fill(fresh[:, None, None, None], 0)
    taps = s["conv_w"].double()
    q, k, v = (torch.zeros((N, B, h, D), dtype=F64, device=DEV) for h in (HK, HK, HV))
    decay, beta = torch.ones((N, B, HV), dtype=F64, device=DEV), torch.zeros((N, B, HV), dtype=F64, device=DEV)
    at = 0
    for b in range(B):
        x = s["mixed"][at:at + n[b]].double()
        past = torch.zeros((3, QKV), dtype=F64, device=DEV) if fresh[b] else conv[slot[b]].t()
        x = torch.cat([past, x])
        conv[slot[b]] = x[-3:].t()
        y = sum(x[i:i + n[b]] * taps[:, i] for i in range(4))
        y = y / (1 + torch.exp(-y))
        for name, first, heads in ((q, 0, HK), (k, HK * D, HK), (v, 2 * HK * D, HV)):
            name[:n[b], b] = y[:, first:first + heads * D].view(n[b], heads, D)
        a = s["a"][at:at + n[b]].double() + s["dt_bias"].double()
        decay[:n[b], b] = torch.exp(-torch.exp(s["A_log"].double()) * torch.nn.functional.softplus(a, threshold=700.0))
        beta[:n[b], b] = 1 / (1 + torch.exp(-s["b"][at:at + n[b]].double()))
        at += n[b]
    q = q / (q.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt() * SCALE
    k = k / (k.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()
    o = torch.zeros((N, B, HV, D), dtype=F64, device=DEV)
    for t in range(N):  # a request whose tokens are over keeps its state: decay 1, beta 0
        kt, qt = k[t].repeat_interleave(2, 1), q[t].repeat_interleave(2, 1)
        S *= decay[t][..., None, None]
        u = beta[t][..., None] * (v[t] - torch.matmul(S, kt[..., None])[..., 0])
        S.addcmul_(u[..., None], kt[..., None, :])
        torch.matmul(S, qt[..., None], out=o[t].unsqueeze(-1))
    h0[slot] = S
    o = torch.cat([o[:n[b], b] for b in range(B)])
    z = s["z"].double().view(T, HV, D)
    out = o / (o.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["norm_w"].double() * z / (1 + torch.exp(-z))
    return [out.view(T, HV * D), conv, h0]
