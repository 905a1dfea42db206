"""The norms around a block in 64 bits from their definition, for the tests (differentiable by autograd)."""
import torch

from delta_reference import far  # noqa: F401


def rows(x, spec, eps):
    if spec is None:
        return x
    kind, weight, bias = tuple(spec) + (None,) * (3 - len(spec))
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    x = x if weight is None else x * weight
    return x if bias is None else x + bias


def residual_norm(block, residual, gate, after, before, scale, activation, eps=1e-6):
    y = rows(block, after, eps)
    if gate is not None:
        y = y * {None: lambda t: t, "sigmoid": torch.sigmoid, "silu": lambda t: t * torch.sigmoid(t)}[activation](gate)
    x = scale * y if residual is None else residual + scale * y
    return x, None if before is None else rows(x, before, eps)


# Tolerances.  fp32: a value passes the sums of a row in at most 2 x 64 steps a lane and a tree (relative error below
# 64 half steps of 2^-24 in 2-norm, less with signs), four of them one after the other in the backward, with factors of
# order one: 4 x 64 x 2^-24 = 1.5e-5.  Results of bf16: one rounding of half a step, 2^-8 at most, on top.
FP32 = 1.5e-5
BF16 = 2.0 ** -8 + FP32


def tolerance(dtype):
    return BF16 if dtype == torch.bfloat16 else FP32


def case(shape, block=torch.float32, stream=None, gate=None, after="rms", before="layer", weights=torch.float32, seed=0,
         biases=True):
    """Inputs of a call on the CPU: (tensors by name, kinds)."""
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    D = shape[-1]
    t = dict(block=(0.5 + randn(*shape)).to(block))
    if stream is not None:
        t["residual"] = (2 * randn(*shape)).to(stream)
    if gate is not None:
        t["gate"] = randn(*gate).to(block)
    for name, kind in (("a", after), ("b", before)):
        if kind is not None:
            t[name + "w"] = (1 + 0.1 * randn(D)).to(weights)
            if kind == "layer" and biases:
                t[name + "b"] = (0.1 * randn(D)).to(weights)
    return t


def spec(t, x, kind):
    return None if kind is None else (kind, t.get(x + "w"), t.get(x + "b"))


def both(t, device, after, before, scale=1.0, activation=None, gradients=True):
    """{name: (result on `device`, wanted in 64 bits)} of a call and its gradients."""
    from fast_transformers_amd.norms import residual_norm as call
    wide = {n: x.double().requires_grad_(gradients) for n, x in t.items()}
    here = {n: x.to(device).requires_grad_(gradients) for n, x in t.items()}
    x, h = call(here["block"], here.get("residual"), here.get("gate"), after=spec(here, "a", after),
                before=spec(here, "b", before), scale=scale, activation=activation)
    want = residual_norm(wide["block"], wide.get("residual"), wide.get("gate"), spec(wide, "a", after),
                         spec(wide, "b", before), scale, activation)
    assert x.dtype == t.get("residual", t["block"]).dtype and (h is None) == (before is None)
    assert h is None or h.dtype == t["block"].dtype
    results = {"x": (x, want[0])}
    if h is not None:
        results["h"] = (h, want[1])
    if gradients:
        gen = torch.Generator().manual_seed(5)
        outs = [o for o in (x, h) if o is not None]
        grads = [torch.randn(o.shape, generator=gen).to(o.dtype) for o in outs]
        got = torch.autograd.grad(outs, list(here.values()), [g.to(device) for g in grads])
        exact = torch.autograd.grad([w for w in want if w is not None], list(wide.values()), [g.double() for g in grads])
        for n, a, b in zip(t, got, exact):
            assert a.dtype == t[n].dtype
            results["grad_" + n] = (a, b)
    return results


def check(results):
    errors = {n: far(a, b) for n, (a, b) in results.items()}
    print({n: "%.2g" % e for n, e in errors.items()}, flush=True)
    for n, (a, _) in results.items():
        assert errors[n] <= tolerance(a.dtype), (n, errors)
