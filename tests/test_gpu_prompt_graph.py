"""The layer node's prompt batches in captured graphs: a graph of a short batch replays as it was after longer ones ran."""
import pytest
import torch
import test_gpu_chunk as chunk
import test_gpu_prompt as prompt

pytestmark = pytest.mark.gpu


def _batch(lens, P, dev, seed):
    h = chunk.make(lens, P, seed, dev)
    g = torch.Generator(device=dev).manual_seed(seed)
    rows = sum(a for a, _ in lens)
    x = torch.randn((rows, 2048), generator=g, device=dev).to(torch.bfloat16)
    key = [torch.arange(k - a, k, device=dev) for a, k in lens]
    loc = torch.cat([h["pt"][b, k // P].long() * P + k % P for b, k in enumerate(key)])
    return h, x, torch.cat(key).to(torch.int32) % 600, loc


def test_a_graph_outlives_longer_batches(dev):
    """The first prompt batch of the node is captured; longer eager ones follow, and memory that they could have freed is
    filled with other values.  Every replay is the eager call, and leaves that memory alone."""
    from bundles_amd.qwen36_layer import engine, layer
    nodes, _, served = prompt._mixer(dev, False)
    P = 16
    batches = [_batch(lens, P, dev, 40 + i) for i, lens in enumerate(([(300, 420)], [(700, 700), (1300, 1500)], [(5000, 5000)]))]
    now = [None]
    view = engine.EngineView()
    view.chunk_view = lambda layer_id, fb: engine.ChunkView(now[0][0]["kc"], now[0][0]["vc"], now[0][0]["pt"], now[0][0]["seqlens"],
                                                            now[0][0]["qsl"], now[0][3], P)
    layer._ChunkScratch._by_device.clear()  # (sets that earlier batches left would be long enough)
    node = layer.prepare(served, engine=view)

    def call(i):
        now[0] = batches[i]
        return node.mixer(batches[i][2], batches[i][1], nodes._batch("extend", batches[i][2]))

    # (a first call of the kernels outside the capture, of a batch that outgrows nothing)
    short = _batch([(200, 290)], P, dev, 50)
    batches.append(short)
    call(3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(0)
    graph.replay()
    torch.cuda.synchronize()
    want = out.clone()
    for i in (1, 2):
        eager = call(i).clone()
        filled = [torch.full((n,), 0x5a, dtype=torch.uint8, device=dev) for n in (1 << 20, 1 << 21, 5 << 20, 132 << 20)]
        for _ in range(2):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert torch.equal(call(0), want)
            assert torch.equal(call(i), eager)
            torch.cuda.synchronize()
        assert all(bool((t == 0x5a).all()) for t in filled)
