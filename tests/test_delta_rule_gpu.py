"""The gated delta rule's kernels against the definition in 64 bits (delta_reference.py, where the tolerances are
derived)."""
import pytest
import torch

import delta_reference as ref
from fast_transformers_amd.delta_rule import gated_delta_rule, gated_delta_step

pytestmark = pytest.mark.gpu

NAMES = ("queries", "keys", "values", "log_decay", "beta", "initial_state")


def check_forward(args, **options):
    dev = [t.cuda() for t in args]
    lengths = options.pop("lengths", None)
    scale = options.setdefault("scale", args[0].shape[3] ** -0.5)
    out, state = gated_delta_rule(*dev, lengths=None if lengths is None else lengths.cuda(), return_state=True, **options)
    want, want_state = ref.rule(*(t.double() for t in args), lengths=lengths, scale=scale,
                                normalize=options.get("normalize", False))
    assert out.dtype == args[2].dtype and state.dtype == torch.float32
    errors = {"out": ref.far(out, want), "state": ref.far(state, want_state)}
    print(errors, flush=True)
    assert errors["out"] <= ref.tolerance(out.dtype), errors
    assert errors["state"] <= ref.FP32, errors
    return out, state


def check_gradients(args, **options):
    dev = [t.cuda().requires_grad_(True) for t in args]
    wide = [t.double().requires_grad_(True) for t in args]
    lengths = options.pop("lengths", None)
    scale = options.setdefault("scale", args[0].shape[3] ** -0.5)
    out, state = gated_delta_rule(*dev, lengths=None if lengths is None else lengths.cuda(), return_state=True, **options)
    want, want_state = ref.rule(*wide, lengths=lengths, scale=scale, normalize=options.get("normalize", False))
    gen = torch.Generator().manual_seed(11)
    go = torch.randn(out.shape, generator=gen).to(out.dtype)
    gs = 0.3 * torch.randn(state.shape, generator=gen)
    got = torch.autograd.grad([out, state], dev, [go.cuda(), gs.cuda()])
    exact = torch.autograd.grad([want, want_state], wide, [go.double(), gs.double()])
    errors = {"out": (ref.far(out, want), out.dtype), "state": (ref.far(state, want_state), state.dtype)}
    for name, x, y, a in zip(NAMES, got, exact, args):
        assert x.dtype == a.dtype and x.shape == a.shape
        errors[name] = (ref.far(x, y), x.dtype)
    print({n: "%.2g" % e for n, (e, _) in errors.items()}, flush=True)
    for name, (e, dtype) in errors.items():
        assert e <= ref.tolerance(dtype), (name, errors)


SHAPES = [  # N, H, Hk, L, E, M
    (1, 1, 1, 64, 32, 16),
    (2, 2, 2, 63, 64, 64),
    (1, 2, 1, 65, 128, 128),
    (1, 2, 2, 9, 64, 80),
    (2, 3, 3, 200, 25, 33),
    (1, 4, 2, 130, 1, 1),
    (1, 2, 2, 129, 100, 7),
    (1, 1, 1, 257, 96, 160),
    (1, 6, 2, 70, 40, 24),
    (1, 1, 1, 66, 128, 512),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype):
    check_forward(ref.inputs(*shape, dtype=dtype, seed=sum(shape)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, dtype):
    check_gradients(ref.inputs(*shape, dtype=dtype, seed=sum(shape)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 4, 2, 130, 64, 64), (2, 2, 1, 150, 128, 48)])
def test_normalized_rows_and_lengths(shape, dtype):
    args = ref.inputs(*shape, dtype=dtype, seed=2, unit=False)
    check_gradients(args, normalize=True)
    for lengths in ([shape[3], 64], [65, 0], [1, 129]):
        check_gradients(args, normalize=True, lengths=torch.tensor(lengths))


@pytest.mark.parametrize("L", [1, 2, 5, 8])
@pytest.mark.parametrize("shape", [(2, 4, 2, 64, 64), (1, 2, 2, 25, 33), (3, 1, 1, 128, 96), (1, 2, 1, 128, 130)])
def test_few_positions(shape, L):
    N, H, Hk, E, M = shape
    for dtype in (torch.float32, torch.bfloat16):
        args = ref.inputs(N, H, Hk, L, E, M, dtype=dtype, seed=L)
        check_forward(args, normalize=True)
        check_forward(args, lengths=torch.arange(N) % (L + 1))
        check_gradients(args)


def test_no_positions():
    args = [t.cuda() for t in ref.inputs(2, 2, 1, 0, 16, 24)]
    out, state = gated_delta_rule(*args, return_state=True)
    assert out.shape == (2, 2, 0, 24) and torch.equal(state, args[5])
    out, state = gated_delta_rule(*args[:5], return_state=True)
    assert not state.any()
    leaves = [t.requires_grad_(True) for t in args]
    out, state = gated_delta_rule(*leaves, return_state=True)
    gs = torch.randn_like(state)
    got = torch.autograd.grad(state, leaves, gs)
    assert torch.equal(got[5], gs)
    empty = ref.inputs(0, 2, 1, 5, 16, 24, device="cuda")
    assert gated_delta_rule(*empty).shape == (0, 2, 5, 24)
