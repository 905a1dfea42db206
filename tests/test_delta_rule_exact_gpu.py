"""The gated delta rule where a result is much smaller than what it is made of, or exactly nothing: gradients of normalised
rows that nearly cancel, rows of few values, positions that write nothing, calls without value heads."""
import pytest
import torch

import delta_reference as ref
from fast_transformers_amd.delta_rule import gated_delta_rule

pytestmark = pytest.mark.gpu

F, B = torch.float32, torch.bfloat16


def gradients(args, go, gs, **options):
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = gated_delta_rule(*leaves, return_state=True, **options)
    return [out.detach(), state.detach(), *torch.autograd.grad([out, state], leaves, [go, gs])]


def wanted(args, go, gs, **options):
    wide = [t.detach().double().cpu().requires_grad_(True) for t in args]
    options.setdefault("scale", args[0].shape[3] ** -0.5)
    out, state = ref.rule(*wide, **options)
    return [out, state, *torch.autograd.grad([out, state], wide, [go.double().cpu(), gs.double().cpu()])]


def along_the_rows(made_of, L, dtype, E=16, M=16, chains=64):
    """A call whose gradient of q, or k, points along the row itself, so that what the normalisation leaves of it is next to
    nothing; (arguments, gradients of the results, which input)."""
    gen = torch.Generator().manual_seed(L)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    k = (randn(1, chains, 1, E) / E ** 0.5).to(dtype).expand(1, chains, L, E).contiguous()
    m = randn(1, chains, 1, M).to(dtype)
    unit = k.double() / (k.double().pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()
    state = (unit[:, :, 0, :, None] * m.double()[:, :, 0, None, :]).float()
    none = torch.zeros_like(state)
    v, go = randn(1, chains, L, M).to(dtype), randn(1, chains, L, M).to(dtype)
    b, forget = torch.rand(1, chains, L, generator=gen) + 0.5, torch.full((1, chains, L), -float("inf"))
    keep, zero = torch.zeros(1, chains, L), torch.zeros(1, chains, L)
    if made_of == "pairs":                # each position reads what it has written itself: dq along k, which is q
        return [k, k.clone(), v, forget, b, none], go, none, 0
    if made_of == "state":                # reads of one state, q times a row: dq along q
        return [k, k.clone(), v, keep, zero, state], go, none, 0
    assert made_of == "written" and L == 1    # the state that is left has a gradient of k times a row: dk along k
    return [k, k.clone(), v, forget, b, none], torch.zeros_like(go), state, 1


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("made_of, L", [("pairs", 1), ("pairs", 70), ("state", 1), ("state", 70), ("written", 1)])
def test_gradients_along_normalised_rows(made_of, L, dtype):
    """What is left of such a gradient is rounding of the whole: that of fp32, whatever the rows' type.  Each part passes a sum of
    16 products (4 half steps of 2^-24 in 2-norm, with signs), a second one of 16 for q . dq, and some dozen single
    roundings (3.5 half steps): below 16 half steps in all.  Results of bf16 are rounded on top, from what is left."""
    args, go, gs, which = along_the_rows(made_of, L, dtype)
    dev = [t.cuda() for t in args]
    got = gradients(dev, go.cuda(), gs.cuda(), normalize=True)[2 + which].double().cpu()
    forgetting = [t.double() for t in args]
    forgetting[3] = forgetting[3].clamp_min(-1000.0)                     # (0 x inf in the definition's own gradient)
    want = wanted(forgetting, go, gs, normalize=True)[2 + which]
    row = args[which].double()
    r = (row.pow(2).sum(-1, keepdim=True) + 1e-6).rsqrt()
    units = [t.double() for t in forgetting]
    for i in (0, 1):
        units[i] = units[i] * (units[i].pow(2).sum(-1, keepdim=True) + 1e-6).rsqrt()
    whole = r * wanted(units, go, gs)[2 + which]                         # before the part along the row is taken away
    assert want.norm() < 1e-4 * whole.norm()
    error, limit = (got - want).norm().item(), 16 * 2.0 ** -24 * whole.norm().item()
    print("error %.3g of the whole, limit %.3g" % (error / whole.norm().item(), 16 * 2.0 ** -24), flush=True)
    assert error <= limit + (2.0 ** -8 * want.norm().item() if dtype == B else 0.0)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("L", [1, 70, 200])
@pytest.mark.parametrize("E", [1, 2, 3, 4, 5, 8, 12, 15])
def test_normalised_rows_of_few_values(E, L, dtype):
    """Of one value nothing but its sign matters: the gradient is 1e-6 / (x^2 + 1e-6) of the whole, not its rounding."""
    args = ref.inputs(2, 4, 2, L, E, 24, dtype=dtype, device="cuda", seed=E, unit=False)
    gen = torch.Generator().manual_seed(E)
    go = torch.randn(args[2].shape, generator=gen).to(dtype).cuda()
    gs = 0.3 * torch.randn(args[5].shape, generator=gen).cuda()
    got, want = gradients(args, go, gs, normalize=True), wanted(args, go, gs, normalize=True)
    errors = [ref.far(a, b) for a, b in zip(got, want)]
    print(["%.2g" % e for e in errors], flush=True)
    for a, e in zip(got, errors):
        assert e <= ref.tolerance(a.dtype), errors


@pytest.mark.parametrize("keep", [False, True], ids=["inference", "training"])
@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("L", [5, 20, 200, 1100])
def test_a_beta_of_zero_writes_nothing(L, dtype, keep):
    q, k, v, g, b, s0 = ref.inputs(1, 2, 1, L, 40, 24, dtype=dtype, device="cuda", seed=L)
    if keep:
        v.requires_grad_(True)
    out, state = gated_delta_rule(q, k, v, g, torch.zeros_like(b), return_state=True)
    assert not out.any() and not state.any()                             # nothing was there, nothing has come
    b = torch.where(torch.arange(L, device="cuda") % 3 == 1, 0.0, b)
    first = gated_delta_rule(q, k, v, g, b, s0, return_state=True)
    with torch.no_grad():
        v[:, :, 1::3] = 1e30 * torch.sign(v[:, :, 1::3])                 # what such a position would write is not looked at
    for x, y in zip(first, gated_delta_rule(q, k, v, g, b, s0, return_state=True)):
        assert torch.equal(x, y)
    tiny = torch.full_like(b, 2.0 ** -100)                               # a write of next to nothing is what it is
    out, state = gated_delta_rule(q, k, v, g, tiny, return_state=True)
    with torch.no_grad():
        full, whole = gated_delta_rule(*(t.double().cpu().float() for t in (q, k, v.sign(), g, tiny)), return_state=True)
    assert state.abs().max() <= 2.0 ** -80 * v.detach().abs().max()      # (at most 1100 writes of 2^-100 v)
    assert whole.abs().max() > 0


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("L", [1, 64, 130])
def test_gradients_where_beta_is_zero(L, normalize):
    args = ref.inputs(2, 4, 2, L, 24, 40, device="cuda", seed=L)
    args[4][:, :, ::2] = 0.0
    args[4][0, 1] = 0.0
    gen = torch.Generator().manual_seed(L)
    go = torch.randn(args[2].shape, generator=gen).cuda()
    gs = 0.3 * torch.randn(args[5].shape, generator=gen).cuda()
    got, want = gradients(args, go, gs, normalize=normalize), wanted(args, go, gs, normalize=normalize)
    errors = [ref.far(a, b) for a, b in zip(got, want)]
    print(["%.2g" % e for e in errors], flush=True)
    assert max(errors) <= ref.FP32, errors
    assert not got[4][:, :, ::2].any()                                   # (values there are not written)


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 24, 40), (1, 2, 1, 1000, 40, 24), (4, 16, 8, 70, 64, 96), (8, 15, 5, 70, 100, 77)])
def test_nothing_comes_of_betas_of_zero(shape, dtype):
    """From no state, and with gradients of the outputs alone, everything but the gradient of beta is exactly zero."""
    args = ref.inputs(*shape, dtype=dtype, device="cuda", seed=1)
    args[4].zero_()
    args[5].zero_()
    go = torch.randn(args[2].shape, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    out, state, gq, gk, gv, gg, gb, gs = gradients(args, go, torch.zeros_like(args[5]), normalize=True)
    for name, t in dict(out=out, state=state, gq=gq, gk=gk, gv=gv, gg=gg).items():
        assert not t.any(), name
    want = wanted(args, go, torch.zeros_like(args[5]), normalize=True)
    assert ref.far(gb, want[6]) <= ref.FP32 and ref.far(gs, want[7]) <= ref.FP32


@pytest.mark.parametrize("L", [0, 5, 70])
def test_no_value_heads(L):
    """Key heads without value heads: empty outputs, gradients of zero."""
    held = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
    del held                                                             # (what the allocator hands out next)
    q, k = (torch.randn(2, 2, L, 8, device="cuda", requires_grad=True) for _ in range(2))
    v = torch.randn(2, 0, L, 4, device="cuda", requires_grad=True)
    g = torch.zeros(2, 0, L, device="cuda", requires_grad=True)
    out, state = gated_delta_rule(q, k, v, g, g, return_state=True)
    assert out.shape == (2, 0, L, 4) and state.shape == (2, 0, 8, 4)
    grads = torch.autograd.grad(out.sum() + state.sum(), [q, k, v, g])
    for t, grad in zip((q, k, v, g), grads):
        assert grad.shape == t.shape and not grad.any()
