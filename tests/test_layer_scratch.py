"""The layer node's buffers as batches grow: a captured graph's stay, the chunk workspace is one a device."""
import types
import weakref

import pytest


@pytest.fixture
def layer(monkeypatch):
    from bundles_amd.qwen36_layer import layer as L

    class Space:
        def __init__(self, *a):
            self.args = a

    for where, name in ((L, "LinearWorkspace"), (L.attn_fused, "Workspace"), (L.attn_fused, "DecodeWorkspace"), (L.attn_fused, "ChunkWorkspace")):
        monkeypatch.setattr(where, name, Space)
    for cls in (L._Scratch, L._ChunkScratch):
        monkeypatch.setattr(cls, "_by_device", {})
    monkeypatch.setattr(L._ChunkScratch, "_chunk_by_device", {}, raising=False)
    return L


@pytest.mark.parametrize("name", ["_Scratch", "_ChunkScratch"])
def test_outgrown_buffers_stay(layer, name):
    cls = getattr(layer, name)
    rows, seen, parts = 0, [], []
    for n in (1, 300, 300, 299, 1000, 1001, 5, 40000, 65535, 65535):
        s = cls.get("gpu 0", n)
        assert s.rows >= n and s.rows >= rows  # (a shorter batch takes the set in use)
        rows = s.rows
        for p in (s.lin2048, s.attn):
            if not any(p is w() for w in parts):
                parts.append(weakref.ref(p))
        if s.rows not in seen:
            seen.append(s.rows)
        del s, p
    assert all(w() is not None for w in parts) and len(parts) == 2 * len(seen)
    assert seen[0] == layer.MAX_TOKENS and all(b >= min(2 * a, 65535) for a, b in zip(seen, seen[1:]))
    assert cls.get("gpu 1", 7).rows == layer.MAX_TOKENS and cls.get("gpu 0", 7).rows == rows


def test_one_chunk_workspace_a_device(layer):
    a = layer._ChunkScratch.get("gpu 0", 10).chunk
    assert layer._ChunkScratch.get("gpu 0", 5000).chunk is a and layer._ChunkScratch.get("gpu 0", 65535).chunk is a
    assert layer._ChunkScratch.get("gpu 1", 10).chunk is not a


def test_engines_that_give_prompt_batches(layer):
    from bundles_amd.qwen36_layer import engine

    class Own(engine.EngineView):
        def chunk_view(self, layer_id, forward_batch):
            return None

    view = engine.EngineView()
    assert not layer._gives_chunks(view) and not layer._gives_chunks(engine.SglangView())
    assert not layer._gives_chunks(types.SimpleNamespace(kv_view=lambda *a: None))
    view.chunk_view = lambda layer_id, fb: None
    assert layer._gives_chunks(view) and layer._gives_chunks(Own())
    assert layer._gives_chunks(types.SimpleNamespace(chunk_view=lambda *a: None))
