"""Sizes that the layers around the gated delta rule take: refused where a layer is made, not at its first call."""
import pytest
import torch

import delta_reference as delta
from fast_transformers_amd.attention import GatedDeltaEncoder, GatedDeltaLayer


@pytest.mark.parametrize("sizes", [(8, 4), (2, 1), (48, 4, 129), (48, 4, 8, 513), (48, 4, 8, 2), (3, 4), (48, 4, 8, 8, 3)])
def test_layers_that_could_not_run_are_not_made(sizes):
    with pytest.raises(ValueError):
        GatedDeltaLayer(*sizes)


def test_models_that_could_not_run_are_not_made():
    with pytest.raises(ValueError, match="d_model"):
        GatedDeltaEncoder(1, 2, 1, d_keys=4, d_values=4)
    with pytest.raises(ValueError, match="d_model"):
        GatedDeltaEncoder(1, 16385, 1, d_keys=4, d_values=4)
    with pytest.raises(ValueError, match="d_values"):
        GatedDeltaEncoder(1, 8, 4)


@pytest.mark.parametrize("sizes", [(3, 1), (12, 4), (5, 2, 1, 3), (6, 4, 128, 512, 1)])
def test_the_least_and_the_most(sizes):
    layer = GatedDeltaLayer(*sizes)
    x = torch.randn(2, 5, sizes[0])
    out, state = layer(x, return_state=True)
    assert torch.isfinite(out).all() and out.shape == x.shape
    step = layer.new_state(2)
    with torch.no_grad():
        last = [layer.step(x[:, i], step) for i in range(5)][-1]
    # (both ways within FP32 of the definition; the norm of a head passes on at most a few times what its row is off by, which the
    # projection of as many heads takes with signs)
    assert delta.far(last, out[:, -1]) <= 8 * delta.FP32 and delta.far(step, state) <= 2 * delta.FP32
