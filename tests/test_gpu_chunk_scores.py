"""The chunk attention at the largest scores: every key's product with a query is 256 * 448^2 or well below it, sums that fp32
holds exactly, so the formula is the mean over the keys of the largest.

Bar: 2^-8 |o| (bf16), (2^-11 + 2^-15) mean |v| (a weight's rounding to f16; sums in fp32)."""
import pytest
import torch
import test_gpu_chunk as chunk

pytestmark = pytest.mark.gpu

BIG, LESS = 0x7e, 0x7d  # 448, 416


@pytest.fixture(scope="module")
def attn():
    from bundles_amd import _lib
    _lib.lib()
    from bundles_amd.qwen36_layer import attn_fused
    return attn_fused


def make(lens, dev, seed, less):
    """Queries and keys of 448; of the keys a share `less` are 416 (weight 0 at these scales), never a request's first."""
    h = chunk.make(lens, 16, seed, dev)
    h["q"][:] = BIG
    h["kc"][:] = BIG
    g = torch.Generator(device=dev).manual_seed(seed)
    low = torch.rand(h["kc"].shape[0], generator=g, device=dev) < less
    low[h["pt"][:, 0].long() * 16] = False
    h["kc"][low] = LESS
    return h, ~low


def formula(h, top):
    out, bar = (torch.zeros(h["q"].shape, dtype=torch.float64, device=h["q"].device) for _ in range(2))
    qsl = h["qsl"].tolist()
    for b, (n, L) in enumerate(h["lens"]):
        key = torch.arange(L, device=out.device)
        slot = h["pt"][b, key // 16].long() * 16 + key % 16
        v, on = chunk.value(h["vc"][slot]), top[slot].double()
        count = on.cumsum(0)[:, None, None]
        for to, w in ((out, v), (bar, v.abs())):
            mean = ((w * on[:, None, None]).cumsum(0) / count)[L - n:]
            to[qsl[b]:qsl[b + 1]] = mean.repeat_interleave(chunk.G, 1)
    return out, 2**-8 * out.abs() + (2**-11 + 2**-15) * bar


@pytest.mark.parametrize("scale", [1 / 16, 0.07, 0.113, 1.0, 30.0, 1e6])
@pytest.mark.parametrize("lens", [[(40, 300)], [(5, 300)], [(1, 5000), (300, 2000), (8, 40)]], ids=["wide", "narrow", "cut"])
@pytest.mark.parametrize("less", [0.0, 0.9])
def test_equal_scores_get_equal_weights(attn, dev, scale, lens, less):
    h, top = make(lens, dev, 7, less)
    print(f"scores of 448 at {scale}", flush=True)
    out = attn.attn_chunk(h["q"], h["kc"], h["vc"], h["pt"], h["seqlens"], h["qsl"], scale, attn.ChunkWorkspace(dev), page_size=16)
    torch.cuda.synchronize()
    want, bar = formula(h, top)
    off = (out.double() - want).abs()
    print(f"scores of 448 at {scale}: {float((off / bar.clamp(min=1e-300)).max()):.3f} of the bar", flush=True)
    assert bool((off <= bar).all())


@pytest.mark.parametrize("scale", [1 / 16, 1.0, 1e6])
def test_a_largest_score_that_comes_late(attn, dev, scale):
    """Keys of 416 first, one of 448 behind them in every 50: the maximum moves among values of millions."""
    h, _ = make([(60, 700)], dev, 8, 0.0)
    key = torch.arange(700, device=dev)
    slot = h["pt"][0, key // 16].long() * 16 + key % 16
    late = key % 50 == 49
    h["kc"][slot[~late]] = LESS
    top = torch.zeros(h["kc"].shape[0], dtype=torch.bool, device=dev)
    top[slot[late]] = True
    out = attn.attn_chunk(h["q"], h["kc"], h["vc"], h["pt"], h["seqlens"], h["qsl"], scale, attn.ChunkWorkspace(dev), page_size=16)
    torch.cuda.synchronize()
    want, bar = formula(h, top)
    assert bool(((out.double() - want).abs() <= bar).all())


@pytest.mark.parametrize("scale", [1 / 16, 1e6])
def test_a_nan_score_is_kept(attn, dev, scale):
    h, _ = make([(40, 300)], dev, 9, 0.0)
    h["kc"][h["pt"][0, 3].long() * 16 + 5, 1, 9] = 0x7f
    out = attn.attn_chunk(h["q"], h["kc"], h["vc"], h["pt"], h["seqlens"], h["qsl"], scale, attn.ChunkWorkspace(dev), page_size=16)
    torch.cuda.synchronize()
    assert bool(out[:, 8:].isnan().all()) and bool(torch.isfinite(out[:, :8]).all())
