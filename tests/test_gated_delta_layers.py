"""The layers around the gated delta rule: the operators in a run, as a model uses them -- against the same model from
the definitions in 64 bits, a prompt in pieces and token by token against the whole, padded batches, gradients."""
import pytest
import torch
import torch.nn.functional as F

import delta_reference as delta
import norm_reference as norm
from fast_transformers_amd.attention import GatedDeltaEncoder
from fast_transformers_amd.masking import LengthMask

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]

# A model of two layers: four blocks one after the other, each within delta.FP32 of its own products, which the next one's
# norms pass on without growth (their factors are of order one): 8 x FP32 in all.
MODEL = 8 * delta.FP32


def model(device, dtype=torch.float32, n_heads=4, n_key_heads=2, seed=0):
    torch.manual_seed(seed)
    m = GatedDeltaEncoder(2, 48, n_heads, d_ff=96, d_keys=16, d_values=24, n_key_heads=n_key_heads, residual_scale=0.7)
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 1:
                p.add_(0.1 * torch.randn(p.shape))
    return m.to(device=device, dtype=dtype)


def definition(m, x, lengths=None):
    """The model from the operators' definitions, float64 on the CPU; parameters by name (leaves)."""
    P = {n: p.detach().double().cpu().requires_grad_(True) for n, p in m.named_parameters()}
    lin = lambda n, t: F.linear(t, P[n + ".weight"], P.get(n + ".bias"))  # noqa: E731
    stream = x
    h = norm.rows(x, ("rms", P["before.0"]), m.eps)
    for i, a in enumerate(m.attentions):
        at = "attentions.%d." % i
        heads = lambda t, n: t.view(*t.shape[:2], n, -1).transpose(1, 2)  # noqa: E731
        q, k = (heads(lin(at + n, h), a.n_key_heads) for n in ("query_projection", "key_projection"))
        v, gate = (heads(lin(at + n, h), a.n_heads) for n in ("value_projection", "gate_projection"))
        g = (-P[at + "log_rate"].exp() * F.softplus(lin(at + "decay_projection", h))).transpose(1, 2)
        b = torch.sigmoid(lin(at + "beta_projection", h)).transpose(1, 2)
        o, _ = delta.rule(q, k, v, g, b, scale=a.d_keys ** -0.5, normalize=True, lengths=lengths)
        o, _ = norm.residual_norm(o, None, gate, ("rms", P[at + "norm_weight"]), None, 1.0, "silu", m.eps)
        out = lin(at + "out_projection", o.transpose(1, 2).flatten(2))
        stream, h = norm.residual_norm(out, stream, None, ("rms", P["after.%d" % (2 * i)]),
                                       ("rms", P["before.%d" % (2 * i + 1)]), m.residual_scale, None, m.eps)
        out = lin("down.%d" % i, F.silu(lin("up.%d" % i, h)))
        stream, h = norm.residual_norm(out, stream, None, ("rms", P["after.%d" % (2 * i + 1)]),
                                       ("rms", P["before.%d" % (2 * i + 2)]), m.residual_scale, None, m.eps)
    return h, P


@pytest.mark.parametrize("device", DEVICES)
def test_model_and_its_gradients_follow_the_definitions(device):
    m = model(device)
    x = torch.randn(3, 90, 48, generator=torch.Generator().manual_seed(1))
    lengths = torch.tensor([90, 64, 7])
    xd = x.to(device).requires_grad_(True)
    h = m(xd, LengthMask(lengths, max_len=90, device=device))
    xw = x.double().requires_grad_(True)
    want, P = definition(m, xw, lengths)
    assert delta.far(h, want) <= MODEL
    go = torch.randn(h.shape, generator=torch.Generator().manual_seed(2))
    got = torch.autograd.grad(h, [xd, *m.parameters()], go.to(device))
    exact = torch.autograd.grad(want, [xw, *P.values()], go.double())
    for n, a, b in zip(["x", *P], got, exact):
        assert delta.far(a, b) <= 4 * MODEL, n   # (the blocks once more, backward, on values that are off themselves)


@pytest.mark.parametrize("device", DEVICES)
def test_a_prompt_in_pieces_and_token_by_token(device):
    m = model(device)
    x = torch.randn(2, 150, 48, generator=torch.Generator().manual_seed(3)).to(device)
    with torch.no_grad():
        whole, last = m(x, return_states=True)
        head, states = m(x[:, :101], return_states=True)
        pieces = [head]
        out, states = m(x[:, 101:106], states=states, return_states=True)   # few positions
        pieces.append(out)
        out, states = m(x[:, 106:140], states=states, return_states=True)
        pieces.append(out)
        pieces += [m.step(x[:, l], states)[:, None] for l in range(140, 150)]
    assert delta.far(torch.cat(pieces, 1), whole) <= 2 * MODEL
    for a, b in zip(states, last):
        assert delta.far(a, b) <= 2 * MODEL
    with torch.no_grad():
        states = m.new_states(2)
        first = m.step(x[:, 0], states)
    assert delta.far(first, whole[:, 0]) <= 2 * MODEL


@pytest.mark.parametrize("device", DEVICES)
def test_half_precision_model_keeps_its_stream_in_fp32(device):
    m = model(device, torch.bfloat16, n_key_heads=4)
    x = torch.randn(2, 70, 48, generator=torch.Generator().manual_seed(4)).to(device=device, dtype=torch.bfloat16)
    h, states = m(x, return_states=True)
    assert h.dtype == torch.bfloat16 and all(s.dtype == torch.float32 for s in states)
    # Every block rounds some eight values on its way (projections, gates, outputs, products), 2^-8 at most each; four blocks of
    # them, their errors added as they are
    want, _ = definition(m, x.double().cpu())
    assert delta.far(h, want) <= 4 * 8 * 2.0 ** -8
    h.float().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())


@pytest.mark.gpu
def test_decoding_in_a_captured_graph():
    m = model("cuda")
    xs = torch.randn(6, 2, 48, device="cuda")
    with torch.no_grad():
        eager = m.new_states(2)
        want = [m.step(x, eager).clone() for x in xs]
        states, x = m.new_states(2), torch.zeros(2, 48, device="cuda")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            m.step(x, states)                     # (allocations and libraries first)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.step(x, states)
        for s in states:
            s.zero_()
        for i in range(6):
            x.copy_(xs[i])
            graph.replay()
            torch.cuda.synchronize()
            torch.ones(1000, device="cuda").sum()  # (the program's own work in between)
            assert torch.equal(out, want[i])
    for a, b in zip(states, eager):
        assert torch.equal(a, b)
