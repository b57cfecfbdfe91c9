"""What TInt8ConnectedLayer takes for its weights and biases."""
import types

import numpy as np
import pytest
import torch

from tensorium_b200 import layers as L

VALUES = [0.5, -1.25, 3.0]


@pytest.mark.parametrize("biases", [np.array(VALUES), np.array(VALUES, np.float32), torch.tensor(VALUES), torch.tensor(VALUES, dtype=torch.float64),
                                    torch.tensor(VALUES, dtype=torch.bfloat16), torch.tensor(VALUES, requires_grad=True), torch.nn.Parameter(torch.tensor(VALUES)), None],
                         ids=["float64 array", "float32 array", "float32", "float64", "bfloat16", "requires grad", "parameter", "none"])
def test_biases(monkeypatch, biases):
    seen = []
    monkeypatch.setattr(L.tokens, "quantize_rows", lambda ctx, w: (w, "scales"))
    monkeypatch.setattr(L.tokens, "int8_connected", lambda ctx, x, w, s, b, act: seen.append(b))
    ctx = types.SimpleNamespace(torch_device=torch.device("cpu"))
    layer = L.TInt8ConnectedLayer(4, 3, weights=torch.ones(3, 4), biases=biases).bind(ctx)
    layer.forward(L.TNNetState(torch.ones(2, 4)))
    b, = seen
    if biases is None:
        assert b is None
    else:
        assert b.dtype == torch.float32 and not b.requires_grad and b.tolist() == VALUES


@pytest.mark.gpu
def test_biases_on_the_gpu(ctx):
    w, b, x = torch.randn(70, 40, device="cuda"), torch.randn(70, device="cuda"), torch.randn(5, 40, device="cuda")
    y = L.TInt8ConnectedLayer(40, 70, weights=w, biases=b).bind(ctx).forward(L.TNNetState(x))
    z = L.TInt8ConnectedLayer(40, 70, weights=w.cpu().numpy(), biases=b.cpu().numpy()).bind(ctx).forward(L.TNNetState(x))
    assert torch.equal(y, z)
