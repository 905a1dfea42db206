"""The gated delta rule and its gradients from the definition, position by position in 64 bits, for the tests."""
import torch


def rule(q, k, v, g, b, s0=None, scale=1.0, normalize=False, lengths=None):
    """(out, state) of float64 tensors, differentiable by autograd."""
    N, H, L, M = v.shape
    group = H // q.shape[1]
    if normalize:
        q, k = (t / (t.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
    q, k = (t.repeat_interleave(group, 1) for t in (q, k))
    S = q.new_zeros((N, H, q.shape[3], M)) if s0 is None else s0
    outs = []
    for l in range(L):
        faded = g[:, :, l].exp()[..., None, None] * S
        z = v[:, :, l] - (k[:, :, l, :, None] * faded).sum(2)
        new = faded + k[:, :, l, :, None] * (b[:, :, l, None] * z)[:, :, None, :]
        out = scale * (q[:, :, l, :, None] * new).sum(2)
        if lengths is not None:
            live = (l < lengths)[:, None, None]
            new = torch.where(live[..., None], new, S)
            out = torch.where(live, out, torch.zeros_like(out))
        S = new
        outs.append(out)
    return (torch.stack(outs, 2) if outs else v.new_zeros((N, H, 0, M))), S


def inputs(N, H, Hk, L, E, M, dtype=torch.float32, seed=0, unit=True, device="cpu", scalars=torch.float32):
    """Queries and keys of length about one, log decays from -0.01 to a few, beta in (0, 1); rows stored (N, L, H, X)."""
    gen = torch.Generator().manual_seed(seed)
    rows = lambda H, X: torch.randn(N, L, H, X, generator=gen).permute(0, 2, 1, 3)  # noqa: E731
    q, k, v = rows(Hk, E), rows(Hk, E), rows(H, M)
    if unit:
        q, k = (torch.nn.functional.normalize(t, dim=-1) for t in (q, k))
    rate = torch.exp(-4 + 4 * torch.rand(H, generator=gen))[None, :, None]
    g = -rate * torch.nn.functional.softplus(torch.randn(N, H, L, generator=gen))
    b = torch.sigmoid(torch.randn(N, H, L, generator=gen))
    s0 = 0.3 * torch.randn(N, H, E, M, generator=gen)
    to = lambda t, d: t.to(d).to(device)  # noqa: E731
    return [to(q, dtype), to(k, dtype), to(v, dtype), to(g, scalars), to(b, scalars), to(s0, torch.float32)]


def far(got, want):
    """2-norm of the difference over that of the wanted values."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    norm = want.norm().item()
    return (got - want).norm().item() / norm if norm else (0.0 if not got.any() else float("inf"))


# Tolerances.  Results of fp32: every one passes sums of at most E + 64 + 64 = 256 products of either sign, whose
# rounding errors in 2-norm are about sqrt(256) half steps (2^-24) of the sum of their squares, some ten such sums one after the
# other (products, the inverse, states of decaying chunks), each times a factor of at most a few (the inverse's
# norm): 10 x 16 x 2^-24 x 2 = 2e-5.  Results of bf16: one rounding, half a step of 2^-8 at most, on top.
FP32 = 2e-5
BF16 = 2.0 ** -8 + FP32


def tolerance(dtype):
    return BF16 if dtype == torch.bfloat16 else FP32
