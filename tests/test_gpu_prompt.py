"""Prompt chunks as they are served: the pages of a batch (paging.plan_pages), its projected rows' front
(attn_fused.attn_front) and the attention over the paged cache (attn_fused.attn_chunk) one after another, and the layer
node's attention mixer over an engine's prompt batches.

Bars: the front's as in test_gpu_front (half a step of the output type and 2^-19 of the magnitudes), the attention's as in
test_gpu_chunk, each against the formula in 64 bits on the operator's own inputs, so that no rounding is counted twice."""
import types

import pytest
import torch
import test_gpu_chunk as chunk
import test_gpu_front as front

pytestmark = pytest.mark.gpu

EPS, SCALE = 1e-6, 1.0 / 16.0


@pytest.fixture(scope="module")
def ops():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import attn_fused, paging
    return attn_fused, paging


class Served:
    """The buffers that a server keeps: caches, request table, free pages, weights; and the batch's own, padded to B and T."""

    def __init__(self, ops, dev, B, T, P, width, pages, axes=None, direct=False, seed=0):
        self.attn, self.paging = ops
        self.P, self.T, self.axes, self.direct = P, T, axes, direct
        g = torch.Generator(device=dev).manual_seed(seed)
        self.kc, self.vc = (torch.full((pages * P, 2, 256), 0x7f, dtype=torch.uint8, device=dev) for _ in range(2))  # NaN
        self.table = torch.zeros((B + 2, width), dtype=torch.int32, device=dev)
        self.free = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        self.req = None if direct else torch.randperm(B + 2, generator=g, device=dev)[:B].to(torch.int32)
        self.cached, self.new = (torch.zeros(B, dtype=torch.int32, device=dev) for _ in range(2))
        # what the attention reads: the pages of the request table's rows, or a slot for each key, written by the plan
        self.pt, self.page = (self.table[:B], P) if direct else (torch.zeros((B, width * P), dtype=torch.int32, device=dev), 1)
        self.plan = self.paging.PagePlan.alloc(B, T, dev)
        self.qw, self.kw = ((torch.randn(256, generator=g, device=dev) * 0.2).to(torch.bfloat16) for _ in range(2))
        self.cos_sin = self.attn.rope_cos_sin(width * P, device=dev)
        self.qkv = torch.zeros((T, 9216), dtype=torch.bfloat16, device=dev)
        self.q = torch.zeros((T, 16, 256), dtype=torch.uint8, device=dev)
        self.gate = torch.zeros((T, 16, 256), dtype=torch.bfloat16, device=dev)
        self.out = torch.zeros((T, 16, 256), dtype=torch.bfloat16, device=dev)
        self.pos = torch.zeros((3, T), dtype=torch.int32, device=dev)
        self.ws = self.attn.ChunkWorkspace(dev)

    def step(self):
        p = self.paging.plan_pages(self.cached, self.new, self.table, self.free, self.T, page_size=self.P, req=self.req,
                                   page_table=None if self.direct else self.pt, whole=True, plan=self.plan)
        pos = p.positions if self.axes is None else self.pos.copy_(p.positions.expand(3, -1))
        self.attn.attn_front(self.qkv, self.qw, self.kw, EPS, self.cos_sin, pos, cache=(self.kc, self.vc, p.out_loc),
                             axes=self.axes, q_dtype=torch.uint8, q=self.q, gate=self.gate)
        self.attn.attn_chunk(self.q, self.kc, self.vc, self.pt, p.seqlens, p.qsl, SCALE, self.ws, page_size=self.page, out=self.out)

    def verify(self, lens, what):
        """The step's outputs: lens (new, keys) of each request; what lies behind the last row is left."""
        n, p = sum(a for a, _ in lens), self.plan
        assert p.used[1] == 0 and p.seqlens.tolist() == [k for _, k in lens]
        rows = torch.cat([torch.arange(k - a, k) for a, k in lens]).to(p.positions)
        assert torch.equal(p.positions[:n], rows) and bool((p.out_loc[n:] == -1).all())
        d = dict(qkv=self.qkv[:n], qw=self.qw, kw=self.kw, cos_sin=self.cos_sin, pos=rows[None].expand(3 if self.axes else 1, -1))
        (wq, mq), wg, (wk, mk), wv = front.formula(d, self.axes.axis_of if self.axes else [0] * 32, self.cos_sin.shape[0])
        front.near(front.value(self.q[:n]), wq, mq, True, f"{what} q")
        assert torch.equal(self.gate[:n].double(), wg)
        front.near(front.value(self.kc[p.out_loc[:n]]), wk, mk, True, f"{what} k")
        front.near(front.value(self.vc[p.out_loc[:n]]), wv, wv.abs() * 0, True, f"{what} v")
        want, bar, mine = chunk.formula(dict(q=self.q, kc=self.kc, vc=self.vc, pt=self.pt, P=self.page, lens=lens, qsl=p.qsl))
        off = (self.out.double() - want).abs()
        print(f"{what}: {float((off / bar.clamp(min=1e-300))[mine].max()):.3f} of the bar", flush=True)
        assert int(mine.sum()) == n and bool((off <= bar)[mine].all())
        assert bool((self.out[n:] == 77).all())

    def fill(self, seed, lens):
        dev = self.qkv.device
        g = torch.Generator(device=dev).manual_seed(seed)
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g, device=dev))
        self.new.copy_(torch.tensor([a for a, _ in lens], dtype=torch.int32))
        self.cached.copy_(torch.tensor([k - a for a, k in lens], dtype=torch.int32))
        self.out.fill_(77)

    def take(self, lens):  # the pages that the step took leave the free list
        used = int(self.plan.used[0])
        self.free = self.free[used:].clone()


STEPS = [[(40, 40), (1, 1), (0, 0), (130, 130)], [(7, 47), (1, 2), (33, 33), (1, 131)], [(1, 48), (90, 92), (1, 34), (0, 131)],
         [(0, 48), (0, 92), (0, 34), (5, 136)]]


@pytest.mark.parametrize("P,axes,direct", [(1, False, False), (16, True, False), (16, False, True), (64, False, True), (64, False, False)])
def test_prompts_in_pieces(ops, dev, P, axes, direct):
    """Four requests over four steps: prompts in pieces, single tokens and idle requests side by side, every key of a
    cache that starts as NaN written by an earlier step or this one."""
    s = Served(ops, dev, 4, 200, P, max(200 // P, 4), 400 // P + 8, ops[0].RopeAxes((11, 11, 10), True) if axes else None, direct)
    for i, lens in enumerate(STEPS):
        s.fill(i, lens)
        s.step()
        torch.cuda.synchronize()
        s.verify(lens, f"P={P} step {i}")
        s.take(lens)


def test_a_step_replays(ops, dev):
    """One captured step over the lengths and pages of each replay: the bits of the eager step."""
    s = Served(ops, dev, 4, 200, 16, 20, 60)
    s.fill(0, STEPS[0])
    s.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.step()
    for i, lens in enumerate(STEPS):
        s.fill(i, lens)
        kept = [t.clone() for t in (s.kc, s.vc, s.table)]
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (s.out, s.q, s.gate, s.kc, s.vc, s.table, s.pt)]
        s.verify(lens, f"replay {i}")
        for t, v in zip((s.kc, s.vc, s.table), kept):
            t.copy_(v)
        s.out.fill_(77)
        s.step()
        torch.cuda.synchronize()
        for a, b in zip(got, (s.out, s.q, s.gate, s.kc, s.vc, s.table, s.pt)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        used = int(s.plan.used[0])
        s.free.copy_(torch.cat([s.free[used:], s.free[:used]]))


def test_pieces_are_the_whole(ops, dev):
    """A prompt in one piece and in three writes the same cache rows and queries, and outputs within their bars."""
    runs = []
    for cuts in ([(190, 190)], [(100, 100), (1, 101), (89, 190)]):
        s = Served(ops, dev, 1, 190, 16, 16, 20, direct=True, seed=3)
        g = torch.Generator(device=dev).manual_seed(9)
        rows = torch.randn((190, 9216), generator=g, device=dev).to(torch.bfloat16)
        out, q = [], []
        for n, k in cuts:
            s.fill(0, [(n, k)])
            s.qkv[:n].copy_(rows[k - n:k])
            s.step()
            torch.cuda.synchronize()
            s.verify([(n, k)], f"piece of {n}")
            out.append(s.out[:n].clone())
            q.append(s.q[:n].clone())
            s.take([(n, k)])
        slot = (s.table[0][torch.arange(190, device=dev) // 16].long() * 16 + torch.arange(190, device=dev) % 16)
        runs.append((torch.cat(q), s.kc[slot], s.vc[slot], torch.cat(out)))
    for a, b in zip(runs[0][:3], runs[1][:3]):
        assert torch.equal(a, b)


# ---- the layer node
def _mixer(dev, axes):
    import test_gpu_nodes as nodes
    from bundles_amd import synth
    ai = synth.attn_inputs(8, dev, seed=31, max_pos=600)
    served = nodes._AttnLayer(nodes._Block(synth.moe_inputs(1, dev, seed=5, E=64)), torch.cat([ai["wqg"], ai["wk"], ai["wv"]]).contiguous(),
                              ai["wo"], ai["q_norm_w"], ai["k_norm_w"], ai["cos_sin"])
    if axes:
        served.rotary_emb.mrope_section, served.rotary_emb.mrope_interleaved = [11, 11, 10], True
    return nodes, ai, served


@pytest.mark.parametrize("axes", [False, True])
def test_layer_node_prompt_chunks(ops, dev, axes):
    """The node's prompt batch is its entries composed by hand, in the engine's cache; rows of no request, the padding
    behind the last one, are the projection of zeros; a view that does not take the batch leaves it to stock."""
    attn, _ = ops
    from bundles_amd.qwen36_layer import engine, glue, layer
    nodes, ai, served = _mixer(dev, axes)
    P, lens = 16, [(150, 150), (1, 200), (40, 333)]
    h = chunk.make(lens, P, 5, dev)
    n, rows = sum(a for a, _ in lens), 196
    g = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn((rows, 2048), generator=g, device=dev).to(torch.bfloat16)
    pos = torch.zeros(rows, dtype=torch.int64, device=dev)
    loc = torch.full((rows,), -1, dtype=torch.int64, device=dev)
    o = 0
    for b, (a, k) in enumerate(lens):
        key = torch.arange(k - a, k, device=dev)
        pos[o:o + a], loc[o:o + a] = key, h["pt"][b, key // P].long() * P + key % P
        o += a
    if axes:
        pos = torch.stack([pos, pos // 2, pos // 3])
    kc, vc = h["kc"].clone(), h["vc"].clone()
    view = engine.EngineView()
    view.chunk_view = lambda layer_id, fb: (engine.ChunkView(kc, vc, h["pt"], h["seqlens"], h["qsl"], loc, P)
                                            if layer_id == 7 and fb.forward_mode.name == "extend" else None)
    node = layer.prepare(served, engine=view)
    out, _ = layer.forward(node, pos, x, None, nodes._batch("extend", pos))
    w = attn.prepare_weights(ai["wqg"], ai["wk"], ai["wv"], ai["wo"])
    qkv = glue.fp8_linear(x, glue.prepare_fp8_weight(torch.cat([ai["wqg"], ai["wk"], ai["wv"]])), glue.LinearWorkspace(rows, 2048, dev))
    q, gate = attn.attn_front(qkv, ai["q_norm_w"], ai["k_norm_w"], EPS, ai["cos_sin"], pos.to(torch.int32), cache=(h["kc"], h["vc"], loc),
                              axes=attn.RopeAxes((11, 11, 10), True) if axes else None, q_dtype=torch.uint8)
    o = torch.zeros((rows, 16, 256), dtype=torch.bfloat16, device=dev)
    attn.attn_chunk(q, h["kc"], h["vc"], h["pt"], h["seqlens"], h["qsl"], SCALE, attn.ChunkWorkspace(dev), P, out=o)
    ref = attn.attn_oproj(o.view(rows, -1), gate.view(rows, -1), w, attn.Workspace(rows, dev))
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), ref.view(torch.int16)) and bool(out[:n].any()) and not bool(out[n:].any())
    assert torch.equal(kc, h["kc"]) and torch.equal(vc, h["vc"])
    assert node.replica.stock_calls == 0
    # other batches, and rows that the positions do not fit, are stock's
    layer.forward(node, pos, x, None, nodes._batch("decode", pos))
    layer.forward(node, pos[..., :-1], x, None, nodes._batch("extend", pos))
    layer.forward(node, pos, x.float(), None, nodes._batch("extend", pos))
    assert node.replica.stock_calls == 3 and served.stock_calls == 0
    plain = layer.prepare(served, engine=types.SimpleNamespace(kv_view=lambda *a: None, gdn_pools=lambda *a: None))
    layer.forward(plain, pos, x, None, nodes._batch("extend", pos))
    assert plain.replica.stock_calls == 1
