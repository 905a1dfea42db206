"""Decayed linear attention: what lies behind a sequence's end is zero whatever the sequence holds, and is not looked at."""
import pytest
import torch

import decay_reference as ref
from fast_transformers_amd.decayed_attention import decayed_attention

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [7, 90, 300])
def test_outputs_behind_the_end_of_a_sequence_without_numbers(device, dtype, L):
    q, k, v, g, s = ref.inputs(3, 2, 2, L, 16, 8, dtype=dtype, device=device)
    lengths = torch.tensor([L - 3, 2, 0], device=device)
    k[0, :, 1], v[1, :, 0], s[1], s[2] = float("nan"), float("inf"), -float("inf"), float("nan")
    for grad in (False, True):
        leaves = [t.detach().clone().requires_grad_(grad) for t in (q, k, v, g, s)]
        out, state = decayed_attention(*leaves, lengths=lengths, return_state=True)
        for n, length in enumerate(lengths.tolist()):
            assert not out[n, :, length:].any()
        assert torch.isnan(state[0]).any() and torch.isnan(state[2]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [7, 90, 300])
def test_gradients_of_outputs_behind_the_end_may_be_anything(device, dtype, L):
    args = ref.inputs(3, 4, 2, L, 16, 8, dtype=dtype, device=device)
    lengths = torch.tensor([L - 3, 2, 0], device=device)
    gen = torch.Generator().manual_seed(2)
    go, gs = torch.randn(args[2].shape, generator=gen).to(dtype).to(device), torch.randn(args[4].shape, generator=gen).to(device)
    behind = torch.arange(L, device=device) >= lengths[:, None]
    spoiled = torch.where(behind[:, None, :, None], float("nan"), go)
    results = []
    for grad_out in (go, spoiled):
        leaves = [t.detach().clone().requires_grad_(True) for t in args]
        out, state = decayed_attention(*leaves, lengths=lengths, return_state=True)
        results.append(torch.autograd.grad([out, state], leaves, [grad_out, gs]))
    assert all(torch.equal(a, b) for a, b in zip(*results))
