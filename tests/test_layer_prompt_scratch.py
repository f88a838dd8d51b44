"""The layer node's buffers of recurrent prompts as batches grow, and which engines hand such batches over."""
import types

import pytest


@pytest.fixture
def layer(monkeypatch):
    from bundles_amd.qwen36_layer import layer as L

    class Space:
        def __init__(self, *a):
            self.args = a

    for where, name in ((L, "LinearWorkspace"), (L.gdn_fused, "PromptWorkspace")):
        monkeypatch.setattr(where, name, Space)
    monkeypatch.setattr(L._PromptScratch, "_by_device", {})
    return L


def test_outgrown_sets_stay(layer):
    seen = []
    for rows, B in ((1, 1), (300, 3), (299, 64), (300, 65), (5, 2), (1000, 200), (65535, 1), (65535, 4000), (1, 1)):
        s = layer._PromptScratch.get("gpu 0", rows, B)
        assert s.rows >= rows and s.B >= B and s.prompt.args == (s.rows, s.B, "gpu 0")
        if s not in seen:
            seen.append(s)
    assert layer._PromptScratch._by_device["gpu 0"] == seen
    assert (seen[0].rows, seen[0].B) == (layer.MAX_TOKENS, 64)
    assert all(b.rows >= a.rows and b.B >= a.B for a, b in zip(seen, seen[1:]))
    assert layer._PromptScratch.get("gpu 1", 7).rows == layer.MAX_TOKENS


def test_engines_that_give_prompts(layer):
    from bundles_amd.qwen36_layer import engine

    class Own(engine.EngineView):
        def gdn_prompt(self, layer_id, forward_batch):
            return None

    assert not layer._gives_prompts(engine.EngineView()) and not layer._gives_prompts(engine.SglangView())
    assert not layer._gives_prompts(types.SimpleNamespace(gdn_pools=lambda *a: None))
    assert layer._gives_prompts(Own()) and layer._gives_prompts(types.SimpleNamespace(gdn_prompt=lambda *a: None))
