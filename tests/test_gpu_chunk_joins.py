"""Calls whose shares of the line are long, so that workgroups that meet in a tile join it themselves, and calls just short of
that: against the formula in 64 bits, and again with the same bits."""
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


@pytest.mark.parametrize("lens", [[(2700, 2700)], [(2900, 2900)], [(5000, 5000)], [(3000, 3300), (1, 9000), (2500, 2500), (5, 40), (700, 4000)]],
                         ids=["short of it", "just past it", "one prompt", "several"])
def test_long_shares(attn, dev, lens):
    h = chunk.make(lens, 16, len(lens) + 60, dev)
    ws = attn.ChunkWorkspace(dev)
    first = chunk.check(attn, h, dev, f"long shares {lens}", ws)
    for _ in range(3):
        assert torch.equal(chunk.run(attn, h, dev, ws), first)
