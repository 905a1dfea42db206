"""Decayed linear attention of many sequences and heads: each route takes as many chains as its own launches have room for."""
import pytest
import torch

import decay_reference as ref
from fast_transformers_amd import _native
from fast_transformers_amd.decayed_attention import decayed_attention, decayed_attention_step

UNSUPPORTED = -2


def plans(N, H, L, M, keep, dtype=0, E=64):
    try:
        return bool(_native.decayed_plan(N, H, H, L, E, M, dtype, keep=keep))
    except RuntimeError as e:
        assert "too many chains" in str(e)
        return False


def test_what_a_route_has_room_for():
    for N, H in ((4096, 32), (8192, 16), (2048, 64), (1 << 16, 16)):
        assert plans(N, H, 1, 64, False) and plans(N, H, 8, 64, False) and plans(N, H, 2000, 64, False)
    # single tokens: workgroups of 1024, or of 256 on states in lots of 16 bytes
    assert plans(1 << 14, (1 << 8) - 1, 1, 63, False) and not plans(1 << 14, 1 << 8, 1, 63, False)
    assert plans((1 << 16) - 1, 1 << 8, 1, 64, False) and not plans(1 << 16, 1 << 8, 1, 64, False)
    assert plans((1 << 13) - 1, 1 << 8, 1, 512, False) and not plans(1 << 13, 1 << 8, 1, 512, False)
    # sequences that keep nothing: workgroups of 512, one a chain
    for dtype in (0, 1):
        assert plans((1 << 15) - 1, 1 << 8, 100, 128, False, dtype) and not plans(1 << 15, 1 << 8, 100, 128, False, dtype)
        assert plans((1 << 13) - 1, 1 << 8, 100, 512, False, dtype) and not plans(1 << 13, 1 << 8, 100, 512, False, dtype)
    # with a backward
    for dtype in (0, 1):
        for E, M in ((64, 64), (128, 128), (8, 512), (128, 8), (1, 1)):
            slices = -(-M // 128)
            assert plans(((1 << 12) - 1) // slices, 1 << 8, 4096, M, True, dtype, E)
            assert plans((1 << 8) // slices, 1 << 6, 250 * 1024, M, True, dtype, E)
            assert not plans(1 << 14, 1 << 9, 2048, M, True, dtype, E)
    assert plans(4096, 32, 1024, 64, True) and not plans(1, 1 << 20, 5000, 64, True)


def test_memory_is_asked_for_what_can_run():
    lib = _native.load()
    for name in ("workspace", "kept", "backward_workspace"):
        f = getattr(lib, "ftc_decayed_attention_%s_bytes" % name)
        assert f(4096, 32, 32, 100, 64, 64, 0) >= 0
        assert f(1 << 13, 1 << 8, 1 << 8, 100, 64, 512, 0) == UNSUPPORTED
    assert lib.ftc_decayed_attention_workspace_bytes(1 << 13, 1 << 9, 1 << 9, 5000, 64, 64, 0) == 0
    assert lib.ftc_decayed_attention_kept_bytes(1 << 13, 1 << 9, 1 << 9, 5000, 64, 64, 0) == UNSUPPORTED


@pytest.mark.gpu
@pytest.mark.parametrize("M", [8, 7])
def test_a_token_of_many_sequences(M):
    q, k, v, g, s = ref.inputs(8200, 16, 16, 1, 8, M, device="cuda")
    want, after = ref.attention(*(t.double() for t in (q, k, v, g, s)), scale=0.25)
    with torch.no_grad():
        got = decayed_attention(q, k, v, g, s, scale=0.25, return_state=True)
    out = decayed_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], s, scale=0.25)
    assert ref.far(out, want[:, :, 0]) <= ref.FP32 and ref.far(s, after) <= ref.FP32
    assert ref.far(got[0], want) <= ref.FP32 and ref.far(got[1], after) <= ref.FP32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_short_sequences(dtype):
    args = ref.inputs(8200, 16, 8, 11, 4, 4, dtype=dtype, device="cuda")
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = decayed_attention(*leaves, return_state=True)
    wide = [t.detach().double().requires_grad_(True) for t in args]
    want, after = ref.attention(*wide, scale=0.5)
    go, gs = torch.randn_like(out), torch.randn_like(state)
    got = torch.autograd.grad([out, state], leaves, [go, gs])
    wanted = torch.autograd.grad([want, after], wide, [go.double(), gs.double()])
    assert ref.far(out, want) <= ref.tolerance(dtype) and ref.far(state, after) <= ref.FP32
    for i, (a, b) in enumerate(zip(got, wanted)):
        assert ref.far(a, b) <= ref.tolerance(a.dtype) + (ref.DECAY if i == 3 else 0)
    with torch.no_grad():
        assert ref.far(decayed_attention(*args), want) <= ref.tolerance(dtype)
