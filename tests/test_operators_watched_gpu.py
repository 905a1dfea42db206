"""The gated delta rule, its step and the norms around a block where a derivative is carried forward, or a call is
traced or transformed: an error or the right answer, never a derivative of zero or a constant."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import delta_reference as delta
from fast_transformers_amd.delta_rule import gated_delta_rule, gated_delta_step
from fast_transformers_amd.norms import residual_norm

pytestmark = pytest.mark.gpu


def rule_inputs(L=20):
    return delta.inputs(1, 2, 1, L, 16, 16, device="cuda")


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("L", [0, 5, 20])
def test_forward_derivatives_of_the_rule_are_refused(L, which, grad):
    args = rule_inputs(L)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward"):
            gated_delta_rule(*args, return_state=True)
        args[which] = fwd.unpack_dual(args[which]).primal
        gated_delta_rule(*args)                     # (a level alone changes nothing)


@pytest.mark.parametrize("which", range(6))
def test_forward_derivatives_of_the_step_are_refused(which):
    q, k, v, g, b, s = rule_inputs(1)
    args = [q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], s]
    before = s.clone()
    with fwd.dual_level():
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward"):
            gated_delta_step(*args)
    assert torch.equal(s, before)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(5))
def test_forward_derivatives_of_the_norms_are_refused(which, grad):
    t = [torch.randn(6, 32, device="cuda") for _ in range(3)] + [torch.ones(32, device="cuda") for _ in range(2)]
    with torch.set_grad_enabled(grad), fwd.dual_level():
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward"):
            residual_norm(t[0], t[1], t[2], after=("rms", t[3]), before=("layer", None, t[4]), activation="silu")


def test_transforms_are_refused():
    args = rule_inputs()
    calls = [(lambda *a: gated_delta_rule(*a).sum(), args),
             (lambda *a: residual_norm(a[0], a[1], before="rms")[1].sum(), [torch.randn(4, 32, device="cuda") for _ in range(2)])]
    q, k, v, g, b, s = rule_inputs(1)
    calls.append((lambda *a: gated_delta_step(*a, s).sum(), [q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0]]))
    for call, given in calls:
        tangents = tuple(torch.ones_like(t) for t in given)
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, tuple(given), tangents)
        with pytest.raises(RuntimeError):
            torch.func.grad(call)(*given)
        with pytest.raises(RuntimeError):
            torch.vmap(call)(*(torch.stack([t, t]) for t in given))


def test_forward_over_backward_is_refused():
    args = [t.requires_grad_(True) for t in rule_inputs()]
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    out, (y, _) = gated_delta_rule(*args), residual_norm(x, after="rms")
    with fwd.dual_level():
        for result, leaves in ((out, args), (y, [x])):
            seed = fwd.make_dual(torch.ones_like(result), torch.ones_like(result))
            with pytest.raises(RuntimeError, match="forward"):
                torch.autograd.grad(result, leaves, seed, retain_graph=True)


def test_traces_see_the_calls():
    args, other = rule_inputs(), delta.inputs(1, 2, 1, 20, 16, 16, device="cuda", seed=3)
    with torch.no_grad():
        traced = torch.jit.trace(lambda *a: gated_delta_rule(*a, normalize=True), tuple(args), check_trace=False)
        assert torch.equal(traced(*other), gated_delta_rule(*other, normalize=True))
        x, y = (torch.randn(2, 6, 32, device="cuda") for _ in range(2))
        traced = torch.jit.trace(lambda a, r: residual_norm(a, r, after="rms", before="layer"), (x[0], x[1]), check_trace=False)
        for a, b in zip(traced(y[0], y[1]), residual_norm(y[0], y[1], after="rms", before="layer")):
            assert torch.equal(a, b)
        q, k, v, g, b, s = rule_inputs(1)
        one = (q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], s)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(lambda *a: gated_delta_step(*a), one, check_trace=False)


@pytest.mark.parametrize("needs", [None, 0, 1, 2, 3, 4])
def test_a_steps_result_has_no_derivative(needs):
    q, k, v, g, b, s = rule_inputs(1)
    args = [q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0]]
    states = [s.clone(), s.clone()]
    with torch.no_grad():
        want = gated_delta_step(*args, states[0])
    if needs is not None:
        args[needs] = args[needs].clone().requires_grad_(True)
    out = gated_delta_step(*args, states[1])
    assert torch.equal(out, want) and torch.equal(*states) and not states[1].requires_grad
    if needs is None:
        assert not out.requires_grad
    else:
        with pytest.raises(RuntimeError, match="cannot be differentiated"):
            (out * out).sum().backward()
    with torch.no_grad():
        assert not gated_delta_step(*args, states[1]).requires_grad


def test_factors_that_would_be_differentiated_are_refused():
    scale = torch.tensor(0.5, device="cuda", requires_grad=True)
    args = rule_inputs()
    x = torch.randn(4, 32, device="cuda")
    with pytest.raises(RuntimeError, match="scale"):
        gated_delta_rule(*args, scale=scale)
    with pytest.raises(RuntimeError, match="scale"):
        residual_norm(x, x, before="rms", scale=scale)
    q, k, v, g, b, s = rule_inputs(1)
    with pytest.raises(RuntimeError, match="scale"):
        gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], s, scale=scale)
    assert torch.equal(gated_delta_rule(*args, scale=scale.detach()), gated_delta_rule(*args, scale=0.5))
    with torch.no_grad():
        assert torch.equal(residual_norm(x, x, scale=scale)[0], residual_norm(x, x, scale=0.5)[0])
