"""The operators of a prompt chunk's way through the attention layer, with their plain forms: the calls
that place a step's new tokens in the paged cache, turn the projection's rows into queries and cache rows,
and attend from the chunk over the cache.

A case is a dict of plain values; its "kind" names the operator:
  pages  paging.plan_pages: row starts, key counts, positions, cache slots and tables of a step, from lengths
  front  attn_fused.attn_front: q / k norm, rotary positions of one or several axes, query and gate rows,
         the new e4m3 rows in the cache
  chunk  attn_fused.attn_chunk: attention of each request's new tokens over its paged e4m3 cache
The model's widths are fixed: 16 query heads over 2 KV heads of 256, the first 64 dims rotated.

Lengths follow from the case alone, values from the seed: request b's length lies between the case's
bounds, spread evenly over the logarithm, in an order that mixes long and short ones.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HQ, HKV, D, ROT = 16, 2, 256, 64
ROWS = 2 * HQ * D + 2 * HKV * D  # a projected row: q and gate of each head, then k, then v
BF, F32, F64, F8, U8, I32, I64 = (torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.uint8,
                                  torch.int32, torch.int64)
EPS, SCALE, MAX_POS = 1e-6, 1.0 / 16.0, 33024
SECTIONS = (11, 11, 10)  # pairs of the time, height and width axes


def listed():
    return [
        # one decode step of a handful of requests: a token each, one-token pages, the tables kept from the
        # step before, so that only the new tokens' entries are written; launch latency is all there is
        dict(name="pages_decode_7", kind="pages", B=7, P=1, cached_min=20, cached_max=3000, new_min=1, new_max=1,
             whole=False),
        # a step that mixes prompt chunks with decoding requests, pages of 16 tokens, tables written whole
        dict(name="pages_mixed_203", kind="pages", B=203, P=16, cached_min=1, cached_max=8191, new_min=1,
             new_max=300, whole=True),
        # a large batch of long conversations whose tables are built anew from pages of 64
        dict(name="pages_long_256", kind="pages", B=256, P=64, cached_min=4000, cached_max=32000, new_min=1,
             new_max=200, whole=True),
        # the front of one decoded token at three axes
        dict(name="front_1", kind="front", T=1, axes=3, interleaved=True, q="bf16"),
        # a prompt with images: contiguous axis sections, e4m3 queries for the chunk attention
        dict(name="front_1777", kind="front", T=1777, axes=3, interleaved=False, q="e4m3"),
        # the largest text chunk: one axis, bf16 queries
        dict(name="front_8192", kind="front", T=8192, axes=1, interleaved=False, q="bf16"),
        # a draft of five tokens over a short context: latency
        dict(name="chunk_1x5", kind="chunk", B=1, P=1, new_min=5, new_max=5, cached_min=295, cached_max=295, q="bf16"),
        # a mixed serving step: decoding requests (one new token) beside prompt chunks, pages of 16
        dict(name="chunk_mixed_24", kind="chunk", B=24, P=16, new_min=1, new_max=509, cached_min=33, cached_max=3500,
             q="e4m3"),
        # the last piece of a long prompt, three requests at once over long contexts, pages of 64
        dict(name="chunk_3x300", kind="chunk", B=3, P=64, new_min=130, new_max=300, cached_min=20000,
             cached_max=32000, q="e4m3"),
        # a chunk of a long prompt after 6000 cached tokens
        dict(name="chunk_1x2048", kind="chunk", B=1, P=1, new_min=2048, new_max=2048, cached_min=6000,
             cached_max=6000, q="e4m3"),
        # eight prompts of a few hundred tokens from an empty cache
        dict(name="chunk_8_prompts", kind="chunk", B=8, P=1, new_min=120, new_max=1000, cached_min=0, cached_max=0,
             q="bf16"),
        # the largest chunk, from an empty cache
        dict(name="chunk_1x8192", kind="chunk", B=1, P=16, new_min=8192, new_max=8192, cached_min=0, cached_max=0,
             q="e4m3"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["pages", "front", "chunk", "chunk"])
    if kind == "pages":
        # 1 .. 512 requests of 0 .. 32000 cached and up to 1000 new tokens, pages of 1 .. 64
        while True:
            B, hi, new = _log_int(rng, 1, 512), _log_int(rng, 16, 32000), _log_int(rng, 1, 1000)
            if B * hi <= 4 << 20 and B * new <= 32768:
                break
        return dict(kind=kind, B=B, P=rng.choice([1, 16, 64]), cached_min=rng.randint(0, hi), cached_max=hi,
                    new_min=rng.randint(1, new), new_max=new, whole=rng.random() < 0.6)
    if kind == "front":
        # 1 .. 8192 tokens, one axis or three, either order of the axes, either type of queries
        axes = rng.choice([1, 3])
        return dict(kind=kind, T=_log_int(rng, 1, 8191), axes=axes, interleaved=axes > 1 and rng.random() < 0.5,
                    q=rng.choice(["bf16", "e4m3"]))
    # 1 .. 64 requests of 1 .. 8000 new tokens over 0 .. 32000 cached ones
    while True:
        B, new = _log_int(rng, 1, 64), _log_int(rng, 1, 8000)
        cached = 0 if rng.random() < 0.2 else _log_int(rng, 1, 32000)
        if B * new * (cached + new / 2) <= 3.0e7 and B * new * (cached + new) <= 6.0e7 and B * (cached + new) <= 1 << 18:
            break
    return dict(kind=kind, B=B, P=rng.choice([1, 16, 64]), new_min=rng.randint(1, new), new_max=new,
                cached_min=rng.randint(0, cached), cached_max=cached, q=rng.choice(["bf16", "e4m3"]))


# ---- lengths --------------------------------------------------------------------------------------------
def _spread(B, lo, hi, turn):
    """B lengths from lo to hi, evenly over log(1 + length), the longest among them."""
    if B == 1:
        return [hi]
    at = [(b * 0.6180339887498949 + turn) % 1.0 for b in range(B)]
    order = sorted(range(B), key=lambda b: at[b])
    out = [0] * B
    for k, b in enumerate(order):
        u = k / (B - 1)
        out[b] = int(round((1 + lo) ** (1 - u) * (1 + hi) ** u)) - 1
    return out


def _lengths(c):
    return (_spread(c["B"], c["cached_min"], c["cached_max"], 0.0), _spread(c["B"], c["new_min"], c["new_max"], 0.37))


# ---- inputs -----------------------------------------------------------------------------------------------
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + salt)
    return g


def _randn(shape, g, std=1.0, dtype=BF):
    return (torch.randn(shape, generator=g, device=DEV, dtype=F32) * std).to(dtype)


def _codes(t):
    return t.clamp(-448, 448).to(F8).view(U8)


def _ints(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def _tables(c, g, spare_rows=3):
    """Pages of every request in random order: the table [rows, width] that holds the cached tokens' pages,
    the requests' rows, the free list (the new tokens' pages first) and the number of slots."""
    P = c["P"]
    cached, new = _lengths(c)
    B, rows = c["B"], c["B"] + spare_rows
    have = [-(-n // P) for n in cached]
    full = [-(-(n + m) // P) for n, m in zip(cached, new)]
    need = sum(full) - sum(have)
    pages = sum(full) + 5
    perm = torch.randperm(pages, generator=g, device=DEV).to(I32)
    width = max(full) + 2
    req = torch.randperm(rows, generator=g, device=DEV)[:B].to(I32)
    table = torch.zeros((rows, width), dtype=I32, device=DEV)
    haves = torch.tensor(have, device=DEV)
    inside = torch.arange(width, device=DEV)[None, :] < haves[:, None]
    part = torch.zeros((B, width), dtype=I32, device=DEV)
    part[inside] = perm[:sum(have)]
    table[req.long()] = part
    free = perm[sum(have):].contiguous()
    assert free.numel() >= need
    return cached, new, req, table, free, pages * P


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind == "pages":
        g = _gen(seed, 1)
        cached, new, req, table, free, _ = _tables(c, g)
        T, width = sum(new), max(a + b for a, b in zip(cached, new)) + 3
        return dict(kind=kind, c=c, cached=_ints(cached), new=_ints(new), req=req, table=table, free=free, T=T,
                    page_table=torch.zeros((c["B"], width), dtype=I32, device=DEV))
    if kind == "front":
        g, T, A = _gen(seed, 2), c["T"], c["axes"]
        inv = 1e7 ** (-torch.arange(0, ROT, 2, dtype=F64, device=DEV) / ROT)
        ang = torch.arange(MAX_POS, dtype=F64, device=DEV)[:, None] * inv
        # text runs on all axes alike; an image's tokens share a time and have a row and a column
        start = int(torch.randint(0, MAX_POS - T, (1,), generator=g, device=DEV))
        pos = (start + torch.arange(T, dtype=I32, device=DEV)).repeat(A, 1)
        if A > 1:
            t = torch.arange(T, device=DEV)
            image = (t // 256) % 2 == 1
            first = start + t // 256 * 256
            pos[0] = torch.where(image, first, pos[0]).to(I32)
            pos[1] = torch.where(image, first + t % 256 // 16, pos[1]).to(I32)
            pos[2] = torch.where(image, first + t % 16, pos[2]).to(I32)
        slots = T + 37
        return dict(kind=kind, c=c, qkv=_randn((T, ROWS), g, 1.5), qw=_randn((D,), g, 0.1), kw=_randn((D,), g, 0.1),
                    cos_sin=torch.cat([ang.cos(), ang.sin()], dim=1).to(F32), pos=pos.contiguous(),
                    out_loc=torch.randperm(slots, generator=g, device=DEV)[:T].contiguous(),
                    kc=torch.zeros((slots, HKV, D), dtype=U8, device=DEV),
                    vc=torch.zeros((slots, HKV, D), dtype=U8, device=DEV))
    g, P = _gen(seed, 3), c["P"]
    cached, new, req, table, free, slots = _tables(c, g)
    # the step's plan, as the page plan leaves it: every request's pages in the batch's order
    full = torch.tensor([-(-(a + b) // P) for a, b in zip(cached, new)], device=DEV)
    have = torch.tensor([-(-a // P) for a in cached], device=DEV)
    off = torch.cumsum(full - have, 0) - (full - have)
    j = torch.arange(table.shape[1], device=DEV)[None, :]
    at = (off[:, None] + j - have[:, None]).clamp(0, free.numel() - 1)
    pt = torch.where(j < have[:, None], table[req.long()], free[at])
    pt = torch.where(j < full[:, None], pt, torch.zeros_like(pt)).contiguous()
    T = sum(new)
    qsl = torch.cat([torch.zeros(1, dtype=I64), torch.cumsum(torch.tensor(new), 0)]).to(I32).to(DEV)
    head = 0.5 + 1.5 * torch.rand((1, HKV, 1), generator=g, device=DEV)
    kc = _codes(torch.randn((slots, HKV, D), generator=g, device=DEV) * head)
    vc = _codes(torch.randn((slots, HKV, D), generator=g, device=DEV) * head)
    q = _randn((T, HQ, D), g, 1.2)
    return dict(kind=kind, c=c, q=_codes(q.float()) if c["q"] == "e4m3" else q, kc=kc, vc=vc, pt=pt, qsl=qsl,
                seqlens=_ints([a + b for a, b in zip(cached, new)]), N=max(new),
                L=max(a + b for a, b in zip(cached, new)), out=torch.zeros((T, HQ, D), dtype=BF, device=DEV))


# ---- the page plan ------------------------------------------------------------------------------------------
def _pages_plain(s):
    c, cached, new, req, table, free = s["c"], s["cached"].long(), s["new"].long(), s["req"].long(), s["table"], s["free"]
    P, T, pt = c["P"], s["T"], s["page_table"]
    zero = torch.zeros(1, dtype=I64, device=DEV)
    qsl = torch.cat([zero, torch.cumsum(new, 0)])
    seqlens = cached + new
    have = (cached + P - 1) // P
    need = (seqlens + P - 1) // P - have
    ends = torch.cumsum(need, 0)
    off = ends - need
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(qsl, t, right=True) - 1
    pos = cached[b] + t - qsl[b]
    j = pos // P
    fresh = j >= have[b]
    page = torch.where(fresh, free[(off[b] + j - have[b]).clamp(0, free.numel() - 1)], table[req[b], j])
    table[req[b], j] = page  # a page's tokens write the same number
    out_loc = page.long() * P + pos % P
    i = torch.arange(pt.shape[1], device=DEV)[None, :]
    keys = table[req][:, (i[0] // P).clamp(max=table.shape[1] - 1)] * P + (i % P).to(I32)
    first = 0 if c["whole"] else cached[:, None]
    pt.copy_(torch.where((i >= first) & (i < seqlens[:, None]), keys, pt))
    used = torch.stack([ends[-1], torch.zeros_like(ends[-1])])
    return [qsl.to(I32), seqlens.to(I32), pos.to(I32), out_loc, table, pt, used.to(I32)]


def _pages_own(s):
    from bundles_amd.qwen36_layer import paging
    c = s["c"]
    if "plan" not in s:
        s["plan"] = paging.PagePlan.alloc(c["B"], s["T"], DEV)
    p = paging.plan_pages(s["cached"], s["new"], s["table"], s["free"], s["T"], page_size=c["P"], req=s["req"],
                          page_table=s["page_table"], whole=c["whole"], plan=s["plan"])
    return [p.qsl, p.seqlens, p.positions, p.out_loc, s["table"], s["page_table"], p.used]


# ---- the front ------------------------------------------------------------------------------------------------
def _axis_of(c):
    """The axis whose position turns pair i (32 pairs)."""
    if c["axes"] == 1:
        return [0] * 32
    if c["interleaved"]:
        return [i % 3 if i % 3 and i < 3 * SECTIONS[i % 3] else 0 for i in range(32)]
    return [0] * SECTIONS[0] + [1] * SECTIONS[1] + [2] * SECTIONS[2]


def _front_math(s, t):
    """q, gate, k, v of the definition in type t, unrounded."""
    x = s["qkv"].to(t)
    T = x.shape[0]
    qg = x[:, :2 * HQ * D].view(T, HQ, 2, D)
    kv = x[:, 2 * HQ * D:].view(T, 2, HKV, D)
    pair = torch.arange(ROT // 2, device=DEV)
    at = s["pos"][torch.tensor(_axis_of(s["c"]), device=DEV)].long().clamp(0, s["cos_sin"].shape[0] - 1).t()
    cos = s["cos_sin"][at, pair].to(t)[:, None, :]
    sin = s["cos_sin"][at, ROT // 2 + pair].to(t)[:, None, :]

    def turned(h, w):
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * (1 + w.to(t))
        a, b = y[..., :ROT // 2], y[..., ROT // 2:ROT]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., ROT:]], dim=-1)

    return turned(qg[:, :, 0], s["qw"]), qg[:, :, 1], turned(kv[:, 0], s["kw"]), kv[:, 1]


def _front_plain(s):
    q, gate, k, v = _front_math(s, F32)
    kc, vc, loc = s["kc"], s["vc"], s["out_loc"]
    kc[loc] = _codes(k)
    vc[loc] = _codes(v)
    q = _codes(q).view(F8) if s["c"]["q"] == "e4m3" else q.to(BF)
    return [q, gate.to(BF), kc.view(F8), vc.view(F8)]


def _front_own(s):
    from bundles_amd.qwen36_layer import attn_fused
    c = s["c"]
    if "axes" not in s:
        s["axes"] = attn_fused.RopeAxes(SECTIONS, c["interleaved"]) if c["axes"] > 1 else None
    q, gate = attn_fused.attn_front(s["qkv"], s["qw"], s["kw"], EPS, s["cos_sin"], s["pos"] if c["axes"] > 1 else s["pos"][0],
                                    cache=(s["kc"], s["vc"], s["out_loc"]), axes=s["axes"],
                                    q_dtype=U8 if c["q"] == "e4m3" else BF)
    return [q.view(F8) if c["q"] == "e4m3" else q, gate, s["kc"].view(F8), s["vc"].view(F8)]


# ---- the chunk's attention --------------------------------------------------------------------------------------
def _chunk_plain(s):
    P, pt, seqlens, qsl, N, L = s["c"]["P"], s["pt"], s["seqlens"].long(), s["qsl"].long(), s["N"], s["L"]
    B, T = pt.shape[0], s["q"].shape[0]
    n = qsl[1:] - qsl[:-1]
    key = torch.arange(L, device=DEV)
    slot = pt[:, key // P].long() * P + key % P
    k = s["kc"][slot].view(F8).to(F32).permute(0, 2, 3, 1).contiguous()  # [B, 2, 256, L]
    v = s["vc"][slot].view(F8).to(F32).permute(0, 2, 1, 3).contiguous()  # [B, 2, L, 256]
    i = torch.arange(N, device=DEV)
    rows = s["q"][(qsl[:-1, None] + i).clamp(max=T - 1)]  # [B, N, 16, 256]
    q = rows.view(F8).to(F32) if s["q"].dtype == U8 else rows.to(F32).clamp(-448, 448).to(F8).to(F32)
    q = q.view(B, N, HKV, HQ // HKV, D).permute(0, 2, 3, 1, 4).reshape(B, HKV, HQ // HKV * N, D)
    p = torch.matmul(q, k).mul_(SCALE).view(B, HKV, HQ // HKV, N, L)
    last = (seqlens - n)[:, None] + i  # [B, N]: the last key that each row sees
    p.masked_fill_(~(key <= last[:, :, None])[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    w = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, HKV, -1, L), v).view(B, HKV, HQ // HKV, N, D).div_(w)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(qsl, t, right=True) - 1
    out = o.permute(0, 3, 1, 2, 4)[b, t - qsl[b]]  # [T, 2, 8, 256]
    return out.reshape(T, HQ, D).to(BF)


def _chunk_own(s):
    from bundles_amd.qwen36_layer import attn_fused
    if "ws" not in s:
        s["ws"] = attn_fused.ChunkWorkspace(DEV)
    return attn_fused.attn_chunk(s["q"], s["kc"], s["vc"], s["pt"], s["seqlens"], s["qsl"], SCALE, s["ws"],
                                 page_size=s["c"]["P"], out=s["out"])


def run(state):
    kind = state["kind"]
    if kind == "pages":
        return _pages_own(state) if own else _pages_plain(state)
    if kind == "front":
        return _front_own(state) if own else _front_plain(state)
    return _chunk_own(state) if own else _chunk_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    c, kind = case, case["kind"]
    if kind == "front":
        T = c["T"]
        q = HQ * D * (1 if c["q"] == "e4m3" else 2)
        per = 2 * ROWS + 8 + 4 * c["axes"] + q + 2 * HQ * D + 2 * HKV * D
        return {"bytes": T * per, "flops": T * (HQ + HKV) * (5 * D + 3 * ROT)}
    cached, new = _lengths(c)
    P, B, T = c["P"], c["B"], sum(new)
    if kind == "pages":
        keys = sum(cached) + T if c["whole"] else T
        pages = sum(-(-(a + b) // P) for a, b in zip(cached, new))
        have = sum(-(-a // P) for a in cached)
        read = 12 * B + 4 * (pages if c["whole"] else pages - have)
        return {"bytes": read + 4 * (pages - have) + 8 * B + 12 * T + 4 * keys + 12, "flops": 0}
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(cached, new))
    keys = sum(cached) + T
    q = HQ * D * (1 if c["q"] == "e4m3" else 2)
    return {"bytes": keys * 2 * HKV * D + T * (q + 2 * HQ * D) + 4 * (-(-keys // P) + 2 * B), "flops": pairs * HQ * 4 * D}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "pages":
        return None  # whole numbers
    if s["kind"] == "front":
        T, A = s["qkv"].shape[0], _axis_of(case)
        x = s["qkv"].double()
        out = {}
        for name, first, heads, step, w in (("q", 0, HQ, 2 * D, s["qw"]), ("k", 2 * HQ * D, HKV, D, s["kw"])):
            rows = []
            for h in range(heads):
                y = x[:, first + h * step:first + h * step + D].clone()
                y /= (y.pow(2).sum(1, keepdim=True) / D + EPS).sqrt()
                y *= 1 + w.double()
                for i in range(ROT // 2):
                    cs = s["cos_sin"][s["pos"][A[i]].long()].double()
                    a, b = y[:, i].clone(), y[:, i + ROT // 2].clone()
                    y[:, i] = a * cs[:, i] - b * cs[:, i + ROT // 2]
                    y[:, i + ROT // 2] = a * cs[:, i + ROT // 2] + b * cs[:, i]
                rows.append(y)
            out[name] = torch.stack(rows, 1)
        gate = torch.stack([x[:, h * 2 * D + D:(h + 1) * 2 * D] for h in range(HQ)], 1)
        v = x[:, 2 * HQ * D + HKV * D:].reshape(T, HKV, D)
        caches = []
        for rows in (out["k"], v):
            cache = torch.zeros(s["kc"].shape, dtype=F64, device=DEV)
            cache[s["out_loc"]] = rows.clamp(-448, 448)
            caches.append(cache)
        q = out["q"].clamp(-448, 448) if case["q"] == "e4m3" else out["q"]
        return [q, gate, *caches]
    P, B = case["P"], case["B"]
    out = torch.zeros(s["out"].shape, dtype=F64, device=DEV)
    qsl, lens = s["qsl"].tolist(), s["seqlens"].tolist()
    for b in range(B):
        t0, t1, L = qsl[b], qsl[b + 1], lens[b]
        pages = s["pt"][b, :-(-L // P)].long()
        slot = (pages[:, None] * P + torch.arange(P, device=DEV)).reshape(-1)[:L]
        k, v = s["kc"][slot].view(F8).double(), s["vc"][slot].view(F8).double()
        for a in range(t0, t1, 1024):
            e = min(a + 1024, t1)
            q = s["q"][a:e]
            q = q.view(F8).double() if q.dtype == U8 else q.float().clamp(-448, 448).to(F8).double()
            seen = L - (t1 - t0) + torch.arange(a - t0, e - t0, device=DEV)
            hide = torch.arange(L, device=DEV)[None, :] > seen[:, None]
            for h in range(HQ):
                z = (q[:, h] @ k[:, h // (HQ // HKV)].t()) * SCALE
                z = torch.softmax(z.masked_fill(hide, -math.inf), dim=1)
                out[a:e, h] = z @ v[:, h // (HQ // HKV)]
    return out
