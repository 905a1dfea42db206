"""Decayed linear attention: log decays of another shape than a call's are refused, on the CPU and on the GPU."""
import pytest
import torch

import decay_reference as ref
from fast_transformers_amd.decayed_attention import decayed_attention, decayed_attention_step

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N, L", [(2, 9), (1, 9), (2, 1), (3, 70)])
@pytest.mark.parametrize("grad", [False, True])
def test_decays_of_one_sequence_or_position_for_all(device, N, L, grad):
    """(1, H, 1) is neither one of every position nor one for each head, and is not spread over either."""
    q, k, v, g, s = ref.inputs(N, 4, 2, L, 16, 8, device=device)
    for bad in (g[:1, :, :1], g[:, :, :1], g[:1], g.transpose(1, 2), g[..., None], g[0]):
        if bad.shape != g.shape:
            with pytest.raises(RuntimeError, match="log_decay"):
                decayed_attention(q, k, v, bad.detach().requires_grad_(grad), s)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N", [1, 2])
def test_a_steps_decays_of_one_sequence_for_all(device, N):
    q, k, v, g, s = ref.inputs(N, 4, 2, 1, 16, 8, device=device)
    before = s.clone()
    for bad in (g[:1, :, 0], g[:, :1, 0], g, g[0, 0], g[:, :, 0].t()):
        if bad.shape != (N, 4):
            with pytest.raises(RuntimeError, match="log_decay"):
                decayed_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], bad, s)
    assert torch.equal(s, before)
    decayed_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], s)
