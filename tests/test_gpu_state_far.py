"""Rows, slots and logits whose offsets pass 32 bits: the same bits as where they lie near the start."""
import pytest
import torch

import test_gpu_drafts as drafts_test
import test_gpu_gdn_commit as commit_test
import test_gpu_gdn_prompt as prompt_test

pytestmark = pytest.mark.gpu
QKV = 8192


@pytest.fixture(scope="module")
def ops():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import gdn_fused
    from bundles_amd.qwen36_lmhead8 import lmhead8
    return gdn_fused, lmhead8


# behind one padded request of 299000 rows by columns, behind five of 59800 by heads
@pytest.mark.parametrize("pads,lens", [([299000], [100, 5]), ([59800] * 5, [100, 5, 100, 100, 90])])
def test_prompt_far_rows_and_slots(ops, dev, pads, lens):
    from bundles_amd.qwen36_layer.glue import linear_rows
    gdn, _ = ops
    print(f"prompt of {lens} behind {sum(pads)} padded rows", flush=True)
    near = prompt_test.inputs(lens, dev, 90, (1,))
    n, gap, P, B, slots = sum(lens), sum(pads), len(pads), len(lens), 2100
    far = {k: near[k] for k in ("conv_w", "A_log", "dt_bias", "norm_w")}
    for k in ("mixed", "z", "a", "b"):
        far[k] = torch.empty((gap + n,) + near[k].shape[1:], dtype=torch.bfloat16, device=dev)
        far[k][:gap] = float("nan")
        far[k][gap:] = near[k]
    far["h0"] = torch.zeros((slots,) + near["h0"].shape[1:], device=dev)
    far["conv_state"] = torch.zeros((slots, QKV, 3), dtype=torch.bfloat16, device=dev)
    at = torch.tensor([2099 - 3 * i for i in range(B)], device=dev)
    far["h0"][at], far["conv_state"][at] = near["h0"][near["state_idx"]], near["conv_state"][near["state_idx"]]
    far["state_idx"] = torch.cat([torch.full((P,), -1, device=dev), at])
    far["qsl"] = torch.cat([torch.tensor([sum(pads[:i]) for i in range(P)], dtype=torch.int32, device=dev), near["qsl"] + gap])
    far["prefix"] = torch.cat([torch.full((P,), 9, dtype=torch.int32, device=dev), near["prefix"]])
    out, oq = torch.full((gap + n, 4096), 3.0, dtype=torch.bfloat16, device=dev), linear_rows(gap + n, 4096, dev)
    want, woq = torch.empty((n, 4096), dtype=torch.bfloat16, device=dev), linear_rows(n, 4096, dev)
    prompt_test.call(gdn, far, out=out, oq=oq)
    prompt_test.call(gdn, near, out=want, oq=woq)
    torch.cuda.synchronize()
    assert not bool(out[:gap].any()) and torch.equal(out[gap:], want)
    assert not bool(oq.scales.view(gap + n, 32)[:gap].any()) and torch.equal(oq.scales.view(gap + n, 32)[gap:], woq.scales.view(n, 32))
    assert torch.equal(oq.codes.view(torch.uint8)[gap:gap + n], woq.codes.view(torch.uint8)[:n])
    used = near["state_idx"]
    assert torch.equal(far["h0"][at], near["h0"][used]) and torch.equal(far["conv_state"][at], near["conv_state"][used])
    rest = torch.ones(slots, dtype=torch.bool, device=dev)
    rest[at] = False
    assert not bool(far["h0"][rest].any()) and not bool(far["conv_state"][rest].any())


def test_drafts_far_rows(ops, dev):
    """2048 requests of 8 rows of 151936, 5 GB of logits: the last ones as in a call of their own."""
    _, lm = ops
    B, T, V, last = 2048, 8, 151936, 3
    print("drafts of 2048 requests", flush=True)
    x = torch.zeros((B * T, V), dtype=torch.bfloat16, device=dev)
    y, d, u, heat, _ = drafts_test.inputs(last, T, V, dev, 91)
    x[-last * T:] = y
    drafts = torch.full((B, T - 1), 5, dtype=torch.int32, device=dev)
    nums, heats = torch.full((B, T), 0.5, device=dev), torch.ones(B, device=dev)
    drafts[-last:], nums[-last:], heats[-last:] = d, u, heat
    tok, n = lm.verify_drafts(x, drafts, nums, lm.VerifyWorkspace(B, T, V, dev), temperature=heats)
    want, wn = lm.verify_drafts(y, d, u, lm.VerifyWorkspace(last, T, V, dev), temperature=heat)
    assert torch.equal(tok[-last:], want) and torch.equal(n[-last:], wn)
    # even rows: a draft of weight 1 / V is refused, the token is the one at half of the rest
    assert bool((n[:-last] == 1).all()) and bool((tok[:-last, 0] == V // 2).all()) and bool((tok[:-last, 1:] == -1).all())


def test_commit_far_slots(ops, dev):
    gdn, _ = ops
    print("commit of far slots", flush=True)
    f = commit_test.pools(3, 4, dev, 92, wp=14)
    want = commit_test.plain(f, 4)
    far = dict(f)
    slots = 2100
    for k, idx in (("h0", "state_idx"), ("conv_state", "state_idx"), ("d_ring", "replay_idx"), ("dlo_ring", "replay_idx"),
                   ("k_ring", "replay_idx"), ("klo_ring", "replay_idx"), ("g_ring", "replay_idx"), ("window", "win_idx"),
                   ("write_pos", "replay_idx"), ("cache_base", "replay_idx")):
        far[k] = torch.zeros((slots,) + f[k].shape[1:], dtype=f[k].dtype, device=dev)
        far[k][2097:2100] = f[k][f[idx]]
    for idx in ("state_idx", "replay_idx", "win_idx"):
        far[idx] = torch.tensor([2097, 2098, 2099], device=dev)
    commit_test.commit(gdn, far, 4)
    torch.cuda.synchronize()
    s, r = f["state_idx"].cpu(), f["replay_idx"].cpu()
    assert torch.equal(far["conv_state"][2097:].cpu(), want["conv_state"][s])
    assert bool(((far["h0"][2097:].cpu().double() - want["h0"][s]).abs() <= want["bound"][s]).all())
    assert torch.equal(far["write_pos"][2097:].cpu(), want["write_pos"][r]) and torch.equal(far["cache_base"][2097:].cpu(), want["cache_base"][r])
    assert not bool(far["h0"][:2097].any()) and not bool(far["conv_state"][:2097].any())
