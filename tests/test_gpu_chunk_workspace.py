"""The chunk attention's workspace: ready for any stream when it is made, made outside captures alone."""
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


def test_ready_for_another_stream(attn, dev):
    """Made behind work that the current stream has yet to do, in memory that held something else: the work and the
    workspace's own launch are done when the constructor returns, so a call on another stream finds it ready."""
    h = chunk.make([(300, 2000), (70, 900)], 16, 1, dev)
    want = chunk.run(attn, h, dev).clone()
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for fill in (0xff, 0x11):
        used = attn.ChunkWorkspace(dev)
        used.buf.fill_(fill)
        del used  # (the allocator gives its memory to the next)
        torch.cuda._sleep(20_000_000)
        ws = attn.ChunkWorkspace(dev)
        assert torch.cuda.current_stream().query()
        out = attn.attn_chunk(h["q"], h["kc"], h["vc"], h["pt"], h["seqlens"], h["qsl"], chunk.SCALE, ws, page_size=16, stream=other)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_not_within_a_capture(attn, dev):
    h = chunk.make([(40, 300)], 16, 2, dev)
    ws, out = attn.ChunkWorkspace(dev), torch.empty_like(h["q"], dtype=torch.bfloat16)
    want = chunk.run(attn, h, dev).clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="before the capture"):
            attn.ChunkWorkspace(dev)
        chunk.run(attn, h, dev, ws, out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        chunk.run(attn, h, dev, ws)
        torch.cuda.synchronize()


def test_a_call_leaves_no_flag(attn, dev):
    """Calls whose workgroups hand partials to one another leave the workspace's flags as the workspace entry does, at zero:
    what an earlier call said of its partials is never there for another to take for its own."""
    groups = torch.cuda.get_device_properties(dev).multi_processor_count
    ws = attn.ChunkWorkspace(dev)
    flags = ws.buf[-(-(-4 * groups // 256) * 256):].view(torch.int32)[:groups]
    assert flags.numel() == groups and not bool(flags.any())
    jobs = [chunk.make(lens, 16, 30 + i, dev) for i, lens in enumerate(([(2000, 2500)], [(700, 900)] * 8, [(5, 300)], [(3000, 3000), (1, 9000)]))]
    want = [chunk.run(attn, h, dev).clone() for h in jobs]
    for _ in range(3):
        for h, w in zip(jobs, want):
            out = chunk.run(attn, h, dev, ws)
            torch.cuda.synchronize()
            assert not bool(flags.any()) and torch.equal(out, w)
