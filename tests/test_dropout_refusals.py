"""The dropout behind a block: refusals and kinds of shares, on the CPU and on the GPU."""
import fractions

import numpy
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


@pytest.mark.parametrize("device", DEVICES)
def test_shares_of_any_kind_of_number(device):
    block = torch.ones(64, 64, device=device)
    for p in (numpy.float16(0.25), numpy.float32(0.25), numpy.float64(0.25), fractions.Fraction(1, 4)):
        assert torch.equal(residual_dropout(block, p=p, seed=3), residual_dropout(block, p=0.25, seed=3))
    for p in (0, 1, False, True, numpy.float16(1)):
        assert torch.equal(residual_dropout(block, p=p, seed=3), block * (1 - int(p)))
