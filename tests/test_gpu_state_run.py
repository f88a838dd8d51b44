"""The recurrent state from prompt to accepted drafts: gdn_prompt, then verify steps over the ring (gdn_verify_ring), drafts
verified (verify_drafts) and committed (gdn_ring_commit), as a server runs them; the layer node's recurrent mixer over an
engine's prompt batches; the hybrid node's accept.

Bar of the state after verify steps: their conv rounds tap products and outputs to bf16 and their history reads high parts
(half steps of 2^-8 of values that enter the state a product at a time): 2^-5 of its norm.  A commit one token off would be
off by the state's own size."""
import types

import numpy as np
import pytest
import torch

import test_gpu_drafts as drafts_test
import test_gpu_gdn_commit as commit_test
import test_gpu_gdn_prompt as prompt_test
import test_gpu_nodes as nodes

pytestmark = pytest.mark.gpu
HK, HV, D, QKV, RING = 16, 32, 128, 8192, 16


@pytest.fixture(scope="module")
def ops():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import gdn_fused
    from bundles_amd.qwen36_lmhead8 import lmhead8
    return gdn_fused, lmhead8


def ring_pools(B, T, dev, seed):
    """Pools of B requests on distinct random slots, all of whose contents are leftovers."""
    g = torch.Generator().manual_seed(seed)
    slots, rslots, wslots = B + 2, B + 1, B + 3
    pick = lambda n: torch.randperm(n, generator=g)[:B].to(dev)  # noqa: E731
    nan = float("nan")
    bf = dict(dtype=torch.bfloat16, device=dev)
    return dict(conv_state=torch.full((slots, QKV, 3), nan, **bf), window=torch.full((wslots, QKV, T + 2), nan, **bf),
                h0=torch.full((slots, HV, D, D), nan, device=dev), d_ring=torch.full((rslots, HV, RING, D), nan, **bf),
                dlo_ring=torch.full((rslots, HV, RING, D), nan, **bf), k_ring=torch.full((rslots, HK, RING, D), nan, **bf),
                klo_ring=torch.full((rslots, HK, RING, D), nan, **bf), g_ring=torch.full((rslots, HV, RING), nan, device=dev),
                state_idx=pick(slots), replay_idx=pick(rslots), win_idx=pick(wslots),
                write_pos=torch.zeros(rslots, dtype=torch.int32, device=dev),
                cache_base=torch.full((rslots,), 13, dtype=torch.int32, device=dev))


@pytest.mark.parametrize("T", [1, 4, 5])
def test_prompts_then_drafts(ops, dev, T):
    """Three requests: prompts of 70, 9 and 1 tokens, ten verify steps, each continued from what was accepted, prompts again."""
    gdn, lm = ops
    print(f"run T={T}", flush=True)
    lens, B, L, V = [70, 9, 1], 3, 150, 999
    f = prompt_test.inputs([L] * B, dev, 40 + T, (0, 1, 2))  # every request's tokens, accepted ones and later tries alike
    rows = lambda name, b, lo, hi: f[name][b * L + lo:b * L + hi]  # noqa: E731
    p = ring_pools(B, T, dev, T)
    cut = {n: torch.cat([rows(n, b, 0, lens[b]) for b in range(B)]) for n in ("mixed", "z", "a", "b")}
    gdn.gdn_prompt(cut["mixed"], cut["z"], cut["a"], cut["b"], p["conv_state"], f["conv_w"], f["A_log"], f["dt_bias"], p["h0"],
                   torch.tensor([0, 70, 79, 80], dtype=torch.int32, device=dev), p["state_idx"], f["norm_w"],
                   gdn.PromptWorkspace(80, B, dev), prefix=torch.zeros(B, dtype=torch.int32, device=dev))
    # a ring's slots are finite numbers: an entry of no weight is multiplied, not skipped
    for n in ("d_ring", "dlo_ring", "k_ring", "klo_ring", "g_ring"):
        p[n].zero_()
    ws, qsl = lm.VerifyWorkspace(B, T, V, dev), torch.arange(0, (B + 1) * T, T, dtype=torch.int32, device=dev)
    at, folds = list(lens), 0
    for step in range(10):
        cut = {n: torch.cat([rows(n, b, at[b], at[b] + T) for b in range(B)]) for n in ("mixed", "z", "a", "b")}
        gdn.gdn_verify_ring(cut["mixed"], cut["z"], cut["a"], cut["b"], p["conv_state"], f["conv_w"], p["window"], f["A_log"],
                            f["dt_bias"], p["h0"], p["d_ring"], p["dlo_ring"], p["k_ring"], p["klo_ring"], p["g_ring"], qsl,
                            p["state_idx"], p["replay_idx"], p["win_idx"], p["write_pos"], p["cache_base"], f["norm_w"], T=T)
        x, d, u, heat, _ = drafts_test.inputs(B, T, V, dev, 100 * T + step)
        tokens, counts = lm.verify_drafts(x, d if T > 1 else None, u, ws, temperature=heat)
        before = p["write_pos"].clone()
        gdn.gdn_ring_commit(*(p[n] for n in commit_test.NAMES[:-1]), counts, T=T, room=16 if step == 9 else None)
        folds += int((p["write_pos"] < before).sum())
        n = counts.tolist()
        assert all(1 <= c <= T for c in n) and ((tokens >= 0).sum(1) == counts).all()
        at = [a + c for a, c in zip(at, n)]
        for b in range(B):
            last = rows("mixed", b, max(at[b] - 3, 0), at[b])
            last = torch.cat([last.new_zeros((3 - last.shape[0], QKV)), last])  # (zeros before a request's first token)
            assert torch.equal(p["conv_state"][p["state_idx"][b]], last.t()), (step, b)
    assert folds > 0 or T == 1
    # the last commit left the rings empty, so a prompt can follow: four tokens of one request, sixteen of the others
    assert not p["write_pos"][p["replay_idx"]].any()
    more = [4, 16, 16]
    cut = {n: torch.cat([rows(n, b, at[b], at[b] + more[b]) for b in range(B)]) for n in ("mixed", "z", "a", "b")}
    gdn.gdn_prompt(cut["mixed"], cut["z"], cut["a"], cut["b"], p["conv_state"], f["conv_w"], f["A_log"], f["dt_bias"], p["h0"],
                   torch.tensor([0, 4, 20, 36], dtype=torch.int32, device=dev), p["state_idx"], f["norm_w"],
                   gdn.PromptWorkspace(36, B, dev))
    at = [n + m for n, m in zip(at, more)]
    whole = dict(f, **{n: torch.cat([rows(n, b, 0, at[b]) for b in range(B)]) for n in ("mixed", "z", "a", "b")})
    whole["qsl"] = torch.tensor(np.concatenate([[0], np.cumsum(at)]), dtype=torch.int32, device=dev)
    _, conv, h0 = prompt_test.plain(whole)
    for b in range(B):
        want, got = h0[whole["state_idx"][b]], p["h0"][p["state_idx"][b]].double()
        assert torch.equal(p["conv_state"][p["state_idx"][b]].double(), conv[whole["state_idx"][b]])
        off = float((got - want).norm() / want.norm())
        print(f"request {b}: {at[b]} tokens, state off by {off:.2e}", flush=True)
        assert off < 2.0 ** -5


def test_captured_steps(ops, dev):
    """Verify step, verification and commit in one captured graph, replayed over changing inputs: every replay leaves the pools
    as eager calls leave theirs."""
    gdn, lm = ops
    B, T, V = 5, 4, 700
    print("captured steps", flush=True)
    pools = [ring_pools(B, T, dev, 7) for _ in range(2)]
    for p in pools:
        for t in p.values():
            if t.is_floating_point():
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(8)) * 0.1)
        p["g_ring"].copy_(-p["g_ring"].abs())
    ws = [lm.VerifyWorkspace(B, T, V, dev) for _ in range(2)]
    qsl = torch.arange(0, (B + 1) * T, T, dtype=torch.int32, device=dev)

    def inputs(seed):
        f = prompt_test.inputs([T] * B, dev, seed)
        x, d, u, heat, _ = drafts_test.inputs(B, T, V, dev, seed)
        return dict({k: f[k] for k in ("mixed", "z", "a", "b", "conv_w", "A_log", "dt_bias", "norm_w")}, x=x, d=d, u=u, heat=heat)

    def step(i, p, w):
        out = gdn.gdn_verify_ring(i["mixed"], i["z"], i["a"], i["b"], p["conv_state"], i["conv_w"], p["window"], i["A_log"],
                                  i["dt_bias"], p["h0"], p["d_ring"], p["dlo_ring"], p["k_ring"], p["klo_ring"], p["g_ring"], qsl,
                                  p["state_idx"], p["replay_idx"], p["win_idx"], p["write_pos"], p["cache_base"], i["norm_w"], T=T)
        tokens, counts = lm.verify_drafts(i["x"], i["d"], i["u"], w, temperature=i["heat"])
        gdn.gdn_ring_commit(*(p[k] for k in commit_test.NAMES[:-1]), counts, T=T)
        return out, tokens, counts
    held = inputs(100)
    saved = {k: t.clone() for k, t in pools[0].items()}
    step(held, pools[0], ws[0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = step(held, pools[0], ws[0])
    for k, t in saved.items():
        pools[0][k].copy_(t)
    for n in range(24):
        new = inputs(100 + n)
        for k, t in new.items():
            held[k].copy_(t)
        g.replay()
        torch.cuda.synchronize()
        want = step(new, pools[1], ws[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), n
        assert all(torch.equal(pools[0][k], pools[1][k]) for k in pools[0]), n
    assert int(pools[1]["cache_base"][pools[1]["replay_idx"]].ne(13).sum()) > 0  # rings were folded


@pytest.mark.parametrize("lens", [[5, 20], [100, 1, 60, 9]])
def test_layer_node_gdn_prompt(ops, dev, lens):
    """The recurrent mixer over an engine's prompt batch (25 rows project through the DENSE8 copies, more through the e4m3
    blocks) equals the same entries composed by hand; batches that the engine does not hand over run stock."""
    from bundles_amd import synth
    from bundles_amd.qwen36_layer import engine, formats, glue, layer
    gdn, _ = ops
    n = sum(lens)
    rows = n + (3 if n > 32 else 0)  # (a padded batch)
    print(f"layer node GDN prompt {lens}", flush=True)
    f = prompt_test.inputs(lens, dev, 31, (0,), rows=rows)
    g = synth.gen(dev, 22)
    x = synth.randn((rows, 2048), g, dev)
    w_qkvz, w_ba = synth.randn((12288, 2048), g, dev, 0.02), synth.randn((64, 2048), g, dev, 0.02)
    w_out = synth.randn((2048, 4096), g, dev, 0.02)
    lin = nodes._LinearAttn(f, w_qkvz, w_ba, w_out, layer_id=3)
    served = nodes._GdnLayer(nodes._Block(synth.moe_inputs(1, dev, seed=5, E=64)), lin)
    mine = {k: v.clone() for k, v in f.items()}
    asked = []

    class View(engine.EngineView):
        def gdn_prompt(self, layer_id, forward_batch):
            asked.append(layer_id)
            if not forward_batch.forward_mode.is_extend():
                return None
            return engine.GdnPrompt(mine["conv_state"], mine["h0"], mine["qsl"], mine["state_idx"], mine["prefix"])
    node = layer.prepare(served, engine=View())
    pos = torch.arange(rows, dtype=torch.int32, device=dev)
    mode = types.SimpleNamespace(is_extend=lambda: True, is_decode=lambda: False, is_target_verify=lambda: False)
    batch = types.SimpleNamespace(forward_mode=mode, positions=pos)
    out, _ = layer.forward(node, pos, x, None, batch)
    e = dict(dtype=torch.bfloat16, device=dev)
    mixed, z = torch.empty((rows, 8192), **e), torch.empty((rows, 4096), **e)
    b, a = torch.empty((rows, 32), **e), torch.empty((rows, 32), **e)
    segs = [(0, mixed), (8192, z), (12288, b), (12320, a)]
    core = torch.zeros((rows, 4096), **e)
    f.update(mixed=mixed, z=z, a=a, b=b)
    if rows <= layer.DENSE8_ROWS:
        glue.dense8_linear(x, *formats.quant_dense8(torch.cat([w_qkvz, w_ba])), segments=segs)
        prompt_test.call(gdn, f, out=core)
        ref = glue.dense8_linear(core, *formats.quant_dense8(w_out))
    else:
        glue.fp8_linear(x, glue.prepare_fp8_weight(torch.cat([w_qkvz, w_ba])), glue.LinearWorkspace(rows, 2048, dev), segs)
        prompt_test.call(gdn, f, out=core)
        ref = glue.fp8_linear(core, glue.prepare_fp8_weight(w_out), glue.LinearWorkspace(rows, 4096, dev))
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), ref.view(torch.int16)) and not out[n:].any()
    assert torch.equal(mine["h0"], f["h0"]) and torch.equal(mine["conv_state"], f["conv_state"])
    rl = node.replica.linear_attn
    assert rl.stock_calls == 0 and asked == [3]
    layer.forward(node, pos, x, None, nodes._batch("decode", pos))
    assert rl.stock_calls == 1 and lin.stock_calls == 0


def test_hybrid_accept(ops, dev):
    """A verify step's logits, its drafts accepted, and every recurrent layer's state moved on: tokens by the definition, the
    layers' pools by the commit's."""
    import test_gpu_hybrid as H
    from bundles_amd import synth
    from bundles_amd.qwen36_layer import hybrid
    _, lm = ops
    w = hybrid.make_weights(dev, seed=3, E=H.E, V=H.V)
    st = hybrid.make_state(H.B, H.T, H.CTX, dev, seed=4, gdn_form="ring", ring_wp=10)
    ws = hybrid.HybridWorkspace(H.B, H.T, H.E, dev, snapshots=False)
    x = synth.randn((H.B * H.T, 2048), synth.gen(dev, 5), dev)
    logits = torch.empty((H.B * H.T, H.V), dtype=torch.bfloat16, device=dev)
    ids = hybrid.forward(x, w, st, ws, logits=logits).view(H.B, H.T)
    assert torch.equal(logits.float().argmax(-1).view(H.B, H.T).to(torch.int32), ids)
    drafts = ids[:, :-1].clone()
    drafts[0, 1] = (drafts[0, 1] + 1) % H.V  # greedy: one draft of the first request is refused
    layers = []
    for conv, S, R in zip(st.conv_state, st.S, st.ring):
        f = dict(conv_state=conv, window=R["window"], h0=S, d_ring=R["d"], dlo_ring=R["dlo"], k_ring=R["k"], klo_ring=R["klo"],
                 g_ring=R["g"], state_idx=R["idx"], replay_idx=R["idx"], win_idx=R["idx"], write_pos=R["wp"], cache_base=R["cb"])
        want = torch.tensor([2] + [H.T] * (H.B - 1))
        layers.append((f, commit_test.plain(dict(f, accepted=want), H.T)))
    u = torch.rand((H.B, H.T), generator=torch.Generator().manual_seed(1)).to(dev)
    tokens, counts = hybrid.accept(logits, drafts, u, st, lm.VerifyWorkspace(H.B, H.T, H.V, dev),
                                   temperature=torch.zeros(H.B, device=dev))
    assert counts.tolist() == [2] + [H.T] * (H.B - 1)
    assert tokens[0, :2].tolist() == ids[0, :2].tolist() and bool((tokens[0, 2:] == -1).all())
    assert torch.equal(tokens[1:], ids[1:])
    for f, want in layers:
        f["accepted"] = want["accepted"].to(dev)
        commit_test.check(f, want)
    st.gdn_form = "snapshot"
    with pytest.raises(ValueError, match="ring"):
        hybrid.accept(logits, drafts, u, st, lm.VerifyWorkspace(H.B, H.T, H.V, dev))
