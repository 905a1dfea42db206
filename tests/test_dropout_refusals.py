"""The dropout behind a block: refusals, on the CPU and on the GPU."""
import pytest
import torch

from fast_transformers_amd.dropout import residual_dropout

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(8,), (2, 8)])
@pytest.mark.parametrize("grad", [False, True])
def test_tensors_without_dimensions(device, shape, grad):
    block, one = torch.randn(shape, device=device).requires_grad_(grad), torch.tensor(1.0, device=device)
    for name in ("residual", "bias"):
        with pytest.raises(RuntimeError, match=name):
            residual_dropout(block, p=0.1, seed=1, **{name: one})
