"""Batches that the attention mixer leaves to stock reach it whatever stands in the positions' place."""
import types

import pytest
import torch


@pytest.mark.parametrize("positions", [None, [0, 1, 2], 7, (torch.zeros(3), torch.zeros(3))], ids=["none", "list", "number", "tuple"])
def test_positions_that_are_no_tensor_are_stock_s(positions):
    from bundles_amd.qwen36_layer import engine, layer
    m, got = object.__new__(layer._AttnMixer), []
    m.engine, m.refusal, m.layer_id, m.replica, m.axes, m.max_tokens = engine.EngineView(), None, 7, object(), None, 8
    m.stock = lambda replica, pos, x, fb: got.append((pos, x)) or "stock"
    x = torch.zeros((3, 2048), dtype=torch.bfloat16)
    assert m(positions, x, types.SimpleNamespace()) == "stock" and got[0][0] is positions and got[0][1] is x
