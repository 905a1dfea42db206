"""The gated delta rule on the CPU: the implementation for CPU tensors against the definition, refusals of the Python
entry points and of the C ABI (no GPU needed)."""
import ctypes

import pytest
import torch

import delta_reference as ref
from fast_transformers_amd import _native
from fast_transformers_amd.delta_rule import gated_delta_rule, gated_delta_step


@pytest.mark.parametrize("L", [0, 1, 31, 32, 33, 100])
@pytest.mark.parametrize("normalize", [False, True])
def test_cpu_tensors_follow_the_definition(L, normalize):
    q, k, v, g, b, s0 = ref.inputs(2, 4, 2, L, 8, 5, seed=L, unit=not normalize)
    out, state = gated_delta_rule(q, k, v, g, b, s0, normalize=normalize, return_state=True)
    want, want_state = ref.rule(*(t.double() for t in (q, k, v, g, b, s0)), scale=8 ** -0.5, normalize=normalize)
    assert out.shape == v.shape and out.dtype == v.dtype
    assert ref.far(state, want_state) <= ref.FP32
    assert ref.far(out, want) <= ref.FP32


def test_cpu_gradients_follow_the_definition():
    args = [t.requires_grad_(True) for t in ref.inputs(2, 4, 2, 50, 8, 6, seed=3)]
    wide = [t.detach().double().requires_grad_(True) for t in args]
    lengths = torch.tensor([50, 17])
    out, state = gated_delta_rule(*args, normalize=True, lengths=lengths, return_state=True)
    want, want_state = ref.rule(*wide, scale=8 ** -0.5, normalize=True, lengths=lengths)
    go, gs = torch.randn(out.shape), torch.randn(state.shape)
    got = torch.autograd.grad([out, state], args, [go, gs])
    exact = torch.autograd.grad([want, want_state], wide, [go.double(), gs.double()])
    for x, y in zip(got, exact):
        assert ref.far(x, y) <= ref.FP32


def test_cpu_step_continues_a_sequence():
    q, k, v, g, b, s0 = ref.inputs(2, 4, 2, 7, 8, 6, seed=5)
    want, want_state = ref.rule(*(t.double() for t in (q, k, v, g, b, s0)), scale=8 ** -0.5)
    state = s0.clone()
    outs = [gated_delta_step(q[:, :, l], k[:, :, l], v[:, :, l], g[:, :, l], b[:, :, l], state) for l in range(7)]
    assert ref.far(torch.stack(outs, 2), want) <= ref.FP32
    assert ref.far(state, want_state) <= ref.FP32


def test_masked_rows_are_not_looked_at():
    q, k, v, g, b, s0 = ref.inputs(2, 2, 2, 20, 8, 4, seed=6)
    lengths = torch.tensor([13, 0])
    clean = gated_delta_rule(q, k, v, g, b, s0, lengths=lengths, return_state=True)
    for t in (q, k, v, g, b):
        t[0, :, 13:] = float("nan")
        t[1] = float("inf")
    out, state = gated_delta_rule(q, k, v, g, b, s0, lengths=lengths, return_state=True)
    assert torch.equal(out, clean[0]) and torch.equal(state, clean[1])
    assert not out[0, :, 13:].any() and not out[1].any() and torch.equal(state[1], s0[1])


def _refused(match, **change):
    q, k, v, g, b, s0 = ref.inputs(2, 4, 2, 5, 8, 6)
    args = dict(queries=q, keys=k, values=v, log_decay=g, beta=b, initial_state=s0)
    args.update(change)
    with pytest.raises(RuntimeError, match=match):
        gated_delta_rule(**args)


def test_refusals():
    q, k, v, g, b, s0 = ref.inputs(2, 4, 2, 5, 8, 6)
    _refused("queries and keys", keys=k[:, :, :4])
    _refused("multiple", queries=torch.zeros(2, 3, 5, 8), keys=torch.zeros(2, 3, 5, 8))
    _refused("one type", values=v.bfloat16())
    _refused("float32 or bfloat16", queries=q.half(), keys=k.half(), values=v.half())
    _refused("log_decay must have shape", log_decay=g[:, :2])
    _refused("beta must have shape", beta=b[:, :, :3])
    _refused("beta must be float32", beta=b.double())
    _refused("1 to 128", queries=torch.zeros(2, 2, 5, 129), keys=torch.zeros(2, 2, 5, 129), initial_state=None)
    _refused("1 to 128", values=torch.zeros(2, 4, 5, 513), initial_state=None)
    _refused("state must be", initial_state=s0[:, :, :, :3])
    _refused("state must be", initial_state=s0.double())
    _refused("lengths", lengths=torch.tensor([5, 5, 5]))
    _refused("expected queries", queries=q[:, 0])
    with pytest.raises(RuntimeError, match="state must be"):
        gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], s0[:, :2])
    with pytest.raises(RuntimeError, match="expected queries"):
        gated_delta_step(q, k, v, g, b, s0)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], s0.requires_grad_(True))


def _t4(shape, dtype=0, ptr=256, stride=None):
    st = stride or (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1)
    return _native.Tensor4(ptr, dtype, tuple(shape), tuple(st))


def _call(N=1, H=2, Hk=1, L=100, E=8, M=8, kept=0, **change):
    """Status of a call whose pointers are never read: every one of these is refused on the host."""
    lib = _native.load()
    t = dict(q=_t4((N, Hk, L, E)), k=_t4((N, Hk, L, E)), v=_t4((N, H, L, M)), g=_t4((N, H, L, 1)), b=_t4((N, H, L, 1)),
             s0=None, out=_t4((N, H, L, M)), s1=None)
    t.update(change)
    r = {n: None if x is None else ctypes.byref(x) for n, x in t.items()}
    return lib.ftc_gated_delta_rule(r["q"], r["k"], r["v"], r["g"], r["b"], None, 1.0, 0, r["s0"], r["out"], r["s1"],
                                    None, 0, None, 0, None), _native.last_error()


def test_c_abi_refuses_on_the_host():
    assert _call(q=None)[0] == -1
    assert _call(k=_t4((1, 1, 99, 8)))[0] == -1
    assert _call(H=3, Hk=2)[0] == -1
    assert _call(E=129)[0] == -2 and _call(M=513)[0] == -2
    assert _call(v=_t4((1, 2, 100, 8), dtype=1))[0] == -1
    assert _call(g=_t4((1, 2, 100, 1), dtype=7))[0] == -1
    assert _call(out=_t4((1, 2, 100, 8), ptr=None))[0] == -1
    assert _call(out=_t4((1, 2, 100, 8), stride=(1600, 800, 8, 2)))[0] == -1
    assert _call(v=_t4((1, 2, 100, 8), stride=(8, 8, (1 << 22) + 1, 1)))[0] == -2
    assert _call(s0=_t4((1, 2, 8, 8), dtype=1))[0] == -1
    assert _call(s1=_t4((1, 2, 8, 9)))[0] == -1
    status, message = _call()                       # no workspace
    assert status == -3 and "needs" in message
    lib = _native.load()
    assert lib.ftc_gated_delta_rule_workspace_bytes(1, 2, 1, 8, 8, 8, 0) == 0
    assert lib.ftc_gated_delta_rule_workspace_bytes(1, 2, 1, 9, 8, 8, 0) > 0
    assert lib.ftc_gated_delta_rule_kept_bytes(1, 3, 2, 9, 8, 8, 0) == -1
    assert lib.ftc_gated_delta_rule_backward_workspace_bytes(1 << 20, 1 << 10, 1, 1 << 20, 128, 128, 0) == -2
    assert lib.ftc_gated_delta_rule_kept_bytes(1, 2, 1, 9, 8, 8, 2) == -1
    q, v, g, s = _t4((1, 1, 1, 8)), _t4((1, 2, 1, 8)), _t4((1, 2, 1, 1)), _t4((1, 2, 8, 8), stride=(0, 0, 8, 1))
    args = [ctypes.byref(t) for t in (q, q, v, g, g)]
    assert lib.ftc_gated_delta_step(*args, 1.0, 0, ctypes.byref(s), ctypes.byref(v), None) == -1
    assert "overlap" in _native.last_error()
    assert lib.ftc_gated_delta_step(*args, 1.0, 0, None, ctypes.byref(v), None) == -1


def test_a_state_that_no_position_changed_is_the_callers_no_more():
    q, k, v, g, b, s0 = ref.inputs(1, 2, 2, 1, 8, 8)
    before = s0.clone()
    _, state = gated_delta_rule(*(t[:, :, :0] for t in (q, k, v, g, b)), s0, return_state=True)
    gated_delta_step(*(t[:, :, 0] for t in (q, k, v, g, b)), state)
    assert torch.equal(s0, before) and not torch.equal(state, before)


def test_calls_of_more_workgroups_than_a_launch_has_are_refused():
    lib = _native.load()
    assert lib.ftc_gated_delta_rule_workspace_bytes(1 << 23, 1, 1, 1, 1, 1, _native.FTC_F32) >= 0
    for N, L, M in ((1 << 24, 1, 1), (1 << 22, 1, 512), (1 << 12, 1 << 19, 64)):
        assert lib.ftc_gated_delta_rule_workspace_bytes(N, 1, 1, L, 1, M, _native.FTC_F32) == -2, (N, L, M)
        assert "too many" in _native.last_error()
