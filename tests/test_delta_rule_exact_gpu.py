"""The gated delta rule where a result is much smaller than what it is made of: gradients of normalised rows that nearly
cancel."""
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
