"""The gated delta rule on CPU tensors: normalised rows of few values, masked rows under gradients, calls without value
heads -- against the definition in 64 bits (delta_reference.py)."""
import pytest
import torch

import delta_reference as ref
from fast_transformers_amd.delta_rule import gated_delta_rule


def gradients(args, go, gs, rule=gated_delta_rule, **options):
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = rule(*leaves, **options)
    return [out.detach(), state.detach(), *torch.autograd.grad([out, state], leaves, [go, gs])]


@pytest.mark.parametrize("L", [1, 50])
@pytest.mark.parametrize("E", [1, 2, 3, 7])
def test_normalised_rows_of_few_values(E, L):
    args = ref.inputs(2, 4, 2, L, E, 6, seed=3, unit=False)
    gen = torch.Generator().manual_seed(E)
    go, gs = (torch.randn(t.shape, generator=gen) for t in (args[2], args[5]))
    got = gradients(args, go, gs, normalize=True, return_state=True)
    want = gradients([t.double() for t in args], go.double(), gs.double(), ref.rule, scale=E ** -0.5, normalize=True)
    errors = [ref.far(a, b) for a, b in zip(got, want)]
    assert max(errors) <= ref.FP32, errors
