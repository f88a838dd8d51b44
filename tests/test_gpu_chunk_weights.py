"""Rows of the chunk attention that one key outweighs by far while the others, each next to nothing, count together: a key of
weight 1 among thousands of weight 2^-25 to 2^-32 with larger values.  (A workgroup's weights are relative to the keys that it
walks itself, so it takes a call that gives each a long walk: 2048 tokens over 262144 keys, 131072 keys a workgroup.)

Bar: 2^-8 |o| (bf16), 2^-11 sum p |v| (a weight's rounding to f16) or 2^-32 sum |v| / l (its absolute half step below f16's
normal range, l the sum of weights relative to the largest), (2^-15 + 2^-17) sum p |v| (sums in fp32; scores exact, their
product with the scale, up to 32 binades, within 2^-24 of itself, and the scale's own rounding)."""
import pytest
import torch
import test_gpu_chunk as chunk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import attn_fused
    return attn_fused


@pytest.mark.parametrize("n,L", [(1, 20011), (7, 9001), (300, 3000), (2048, 20011), (2048, 262144)])
@pytest.mark.parametrize("where", ["first", "last", "middle"])
def test_small_weights_count(attn, dev, n, L, where):
    h = chunk.make([(n, L)], 16, n + L, dev)
    g = torch.Generator(device=dev).manual_seed(L)
    key = torch.arange(L, device=dev)
    slot = h["pt"][0, key // 16].long() * 16 + key % 16
    # all of a key's dims alike, queries of 1: score = 16 times the key's value
    k = chunk.codes(-0.25 * torch.rand(L, generator=g, device=dev))
    at = {"first": 0, "last": L - n, "middle": L // 2}[where]  # (a key that all the new tokens see)
    k[at] = 0x39  # 1.125
    h["kc"][slot] = k[:, None, None].expand(L, chunk.HKV, chunk.D)
    v = chunk.codes(8 + 440 * torch.rand((L, chunk.HKV, chunk.D), generator=g, device=dev))
    v[at] = 0xb8  # -1
    h["vc"][slot] = v
    h["q"][:] = 0x38  # 1
    print(f"small weights n={n} L={L} {where}", flush=True)
    out = chunk.run(attn, h, dev)
    torch.cuda.synchronize()
    x = torch.exp(16 * (chunk.value(k) - 1.125))
    val = chunk.value(v)
    worst = 0.0
    for t in sorted({0, n // 2, n - 1}):
        end = L - n + t + 1
        l = x[:end].sum()  # noqa: E741
        o = (x[:end, None, None] * val[:end]).sum(0) / l
        pv = (x[:end, None, None] * val[:end].abs()).sum(0) / l
        bar = 2**-8 * o.abs() + (2**-11 + 2**-15 + 2**-17) * pv + 2**-32 * val[:end].abs().sum(0) / l
        off = (out[t].double() - o.repeat_interleave(chunk.G, 0)).abs()
        worst = max(worst, float((off / bar.repeat_interleave(chunk.G, 0)).max()))
    print(f"small weights n={n} L={L} {where}: {worst:.3f} of the bar", flush=True)
    assert worst <= 1
