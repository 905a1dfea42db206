"""States that a step updates in place: any layout whose rows lie apart, none whose rows share memory (no GPU needed: the C
ABI refuses on the host, before its pointers are read)."""
import ctypes

import pytest
import torch

import delta_reference as ref
from fast_transformers_amd import _native
from fast_transformers_amd.delta_rule import gated_delta_step

N, H, E, M = 2, 3, 4, 5
# strides of (N, H, E), the last dimension's is 1
SHARED = [(0, 20, 5), (60, 0, 5), (60, 20, 0), (60, 20, 4), (60, 19, 5), (59, 20, 5), (20, 20, 5), (10, 20, 5)]
APART = [(60, 20, 5), (64, 21, 5), (20, 40, 5), (5, 40, 10), (60, 5, 15), (1000, 300, 7), (5, 10, 30)]


def step_on_the_host(strides):
    """Status of a call without queries' memory: -1 for both reasons, told apart by the message."""
    t4 = lambda shape, stride: _native.Tensor4(256, 0, shape, stride)  # noqa: E731
    q, v, g = t4((N, H, 1, E), (H * E, E, E, 1)), t4((N, H, 1, M), (H * M, M, M, 1)), t4((N, H, 1, 1), (H, 1, 1, 1))
    s, out = t4((N, H, E, M), (*strides, 1)), t4((N, H, 1, M), (H * M, M, M, 1))
    r = ctypes.byref
    return _native.load().ftc_gated_delta_step(r(q), r(q), r(v), r(g), r(g), 1.0, 0, r(s), r(out), None)


@pytest.mark.parametrize("strides", SHARED)
def test_rows_that_share_memory_are_refused(strides):
    assert step_on_the_host(strides) == -1 and "overlap" in _native.last_error()
    q, k, v, g, b, _ = ref.inputs(N, H, H, 1, E, M)
    state = torch.zeros(2000).as_strided((N, H, E, M), (*strides, 1))
    with pytest.raises(RuntimeError, match="overlap"):
        gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], state)


@pytest.mark.parametrize("strides", APART)
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rows_that_lie_apart(strides, device):
    q, k, v, g, b, s0 = ref.inputs(N, H, H, 1, E, M, device=device)
    memory = torch.full((2000,), 7.0, device=device)
    state = memory.as_strided((N, H, E, M), (*strides, 1))
    state.copy_(s0)
    out = gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], state)
    want, after = ref.rule(*(t.double().cpu() for t in (q, k, v, g, b, s0)), scale=E ** -0.5)
    assert ref.far(out, want[:, :, 0]) <= ref.FP32 and ref.far(state, after) <= ref.FP32
    assert (memory == 7.0).sum() == 2000 - N * H * E * M
