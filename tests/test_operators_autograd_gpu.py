"""The gated delta rule and the norms around a block under autograd: second derivatives are refused, not missed; the
state of a step counts its versions; the norms watched, captured, on other streams, far apart, against differences."""
import pytest
import torch

import delta_reference as delta
import norm_reference as norm
from fast_transformers_amd.delta_rule import gated_delta_rule, gated_delta_step
from fast_transformers_amd.norms import residual_norm

pytestmark = pytest.mark.gpu

F, B = torch.float32, torch.bfloat16


def watched():
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)


@pytest.mark.parametrize("watch", [False, True])
@pytest.mark.parametrize("L", [0, 70])
def test_second_derivatives_of_the_rule_are_refused(watch, L):
    args = [t.requires_grad_(True) for t in delta.inputs(1, 2, 1, L, 16, 16, device="cuda")]
    if watch:
        with watched():
            out, state = gated_delta_rule(*args, return_state=True)
    else:
        out, state = gated_delta_rule(*args, return_state=True)
    grads = torch.autograd.grad(out.square().sum() + state.square().sum(), args, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        (grads[1].square().sum() + grads[5].square().sum()).backward()
    # (a gradient that does not depend on the outputs' values, beside a term that can be differentiated)
    out = gated_delta_rule(*args)
    (grad,) = torch.autograd.grad(out.sum(), args[0], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad((grad * args[0]).sum(), args[0])


@pytest.mark.parametrize("watch", [False, True])
def test_second_derivatives_of_the_norms_are_refused(watch):
    t = {n: x.cuda().requires_grad_(True) for n, x in norm.case((9, 64), F, F, (9, 64), "rms", "layer").items()}
    call = lambda: residual_norm(t["block"], t["residual"], t["gate"], after=norm.spec(t, "a", "rms"),  # noqa: E731
                                 before=norm.spec(t, "b", "layer"))
    if watch:
        with watched():
            x, h = call()
    else:
        x, h = call()
    grads = torch.autograd.grad(x.sum() + h.sum(), list(t.values()), create_graph=True)
    for n, grad in zip(t, grads):
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad((grad * t["block"].detach().flatten()[0]).sum(), t["block"], retain_graph=True)


def test_a_step_counts_the_states_versions():
    q, k, v, g, b, s0 = delta.inputs(2, 2, 2, 1, 16, 16, device="cuda")
    weight = torch.ones_like(s0, requires_grad=True)
    product = (s0 * weight).sum()                      # (saves the state)
    gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], s0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():
        s = torch.zeros_like(s0)
        out = gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], g[:, :, 0], b[:, :, 0], s)
        assert torch.isfinite(out).all() and s.any()


def test_an_input_changed_before_the_backward_is_an_error():
    args = [t.requires_grad_(True) for t in delta.inputs(1, 1, 1, 70, 16, 16, device="cuda")]
    out = gated_delta_rule(*args)
    with torch.no_grad():
        args[1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    x = torch.randn(5, 64, device="cuda", requires_grad=True)
    y, _ = residual_norm(x, after="rms")
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def gradients(t, after, before, go=None):
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items()}
    x, h = residual_norm(leaves["block"], leaves.get("residual"), leaves.get("gate"), after=norm.spec(leaves, "a", after),
                         before=norm.spec(leaves, "b", before), scale=0.5, activation="silu")
    outs = [o for o in (x, h) if o is not None]
    go = go or [torch.cos(torch.arange(o.numel(), device="cuda", dtype=F)).view(o.shape).to(o.dtype) for o in outs]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(leaves.values()), go))


def test_watched_norms():
    t = {n: x.cuda() for n, x in norm.case((3, 40, 64), B, F, (3, 1, 64), "rms", "layer").items()}
    plain = gradients(t, "rms", "layer")
    with watched():
        seen = gradients(t, "rms", "layer")
    assert all(torch.equal(a, b) for a, b in zip(plain, seen))


def test_differences_of_the_norms():
    """Gradients against central differences, in a direction of every input."""
    t = {n: x.cuda() for n, x in norm.case((7, 96), F, F, (7, 96), "layer", "rms").items()}
    grads = gradients(t, "layer", "rms")[2:]
    gen = torch.Generator(device="cuda").manual_seed(2)

    def loss(m):
        outs = residual_norm(m["block"], m["residual"], m["gate"], after=norm.spec(m, "a", "layer"),
                             before=norm.spec(m, "b", "rms"), scale=0.5, activation="silu")
        return sum((o.double() * torch.cos(torch.arange(o.numel(), device="cuda", dtype=F)).view(o.shape)).sum() for o in outs)
    h = 2.0 ** -7
    for n, grad in zip(t, grads):
        d = torch.randn(t[n].shape, generator=gen, device="cuda")
        d = d / d.norm()
        up, down = (loss({**t, n: t[n] + s * h * d}).item() for s in (1, -1))
        # Rounding of 2 x 672 values of order 2, 2^-23 each with random signs and weights of order one: 2 x 37 x 2^-23 / 2h; the
        # third derivative along a unit step is of order 10 (rows of deviation one), h^2 / 6 of it
        assert abs((up - down) / (2 * h) - (grad.double() * d).sum().item()) <= 74 * 2.0 ** -23 / (2 * h) + 10 * h * h / 6, n


def test_norms_of_rows_far_apart():
    """Rows 2^23 elements apart: the last lie 5 GB behind the first."""
    t = {n: x.cuda() for n, x in norm.case((600, 128), B, B, (600, 128), "rms", "rms").items()}
    buffer = torch.zeros((600, 1 << 22), device="cuda", dtype=B)
    far = dict(t)
    for i, n in enumerate(("block", "residual", "gate")):
        view = buffer[:, 128 * i:128 * i + 128]
        view.copy_(t[n])
        far[n] = view
    for a, b in zip(gradients(far, "rms", "rms"), gradients(t, "rms", "rms")):
        assert torch.equal(a, b)


def test_rows_that_are_one_row_and_tensors_used_twice():
    row = torch.randn(1, 1, 96, generator=torch.Generator().manual_seed(1)).cuda().expand(4, 9, 96)
    w = torch.rand(96, device="cuda").add_(0.5).requires_grad_(True)
    leaf = row.detach().requires_grad_(True)
    x, h = residual_norm(leaf, leaf, leaf, after=("rms", w, w), before=("layer", w), activation="sigmoid")
    got = torch.autograd.grad((x.square() + h * x).sum(), [leaf, w])
    lw, ww = leaf.detach().double().cpu().requires_grad_(True), w.detach().double().cpu().requires_grad_(True)
    X, H = norm.residual_norm(lw, lw, lw, ("rms", ww, ww), ("layer", ww), 1.0, "sigmoid")
    want = torch.autograd.grad((X.square() + H * X).sum(), [lw, ww])
    assert norm.far(x, X) <= norm.FP32 and norm.far(h, H) <= norm.FP32
    assert all(norm.far(a, b) <= 2 * norm.FP32 for a, b in zip(got, want))   # (sums of parts that each have their own error)


def test_norms_on_streams_and_in_graphs():
    """Two streams at once; two captured graphs of forward and backward, replayed with eager work between."""
    cases = [{n: x.cuda() for n, x in norm.case((20, 33, 512), B, F, (20, 1, 512), "layer", "rms", seed=s).items()} for s in (1, 2)]
    want = [gradients(t, "layer", "rms") for t in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for i, t in enumerate(cases):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = gradients(t, "layer", "rms")
    torch.cuda.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(x, y))
    held = [{n: x.clone() for n, x in t.items()} for t in cases]
    graphs, outs = [], []
    go = [torch.ones(20, 33, 512, device="cuda"), torch.ones(20, 33, 512, device="cuda", dtype=B)]  # (the graphs read them)
    for t in held:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            gradients(t, "layer", "rms", go)
        torch.cuda.current_stream().wait_stream(stream)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(gradients(t, "layer", "rms", go))
    for turn in range(4):
        new = [{n: x.cuda() for n, x in norm.case((20, 33, 512), B, F, (20, 1, 512), "layer", "rms", seed=10 + 2 * turn + i).items()}
               for i in range(2)]
        for t, values in zip(held, new):
            for n in t:
                t[n].copy_(values[n])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for values, out in zip(new, outs):
            assert all(torch.equal(a, b) for a, b in zip(gradients(values, "layer", "rms", go), out)), turn


def test_nothing_beside_the_rows_is_looked_at():
    """Places between strided rows may hold anything, and a row of NaN stays in its row."""
    wide = torch.full((50, 3, 96), float("nan"), device="cuda")
    wide[:, 1] = torch.randn(50, 96, device="cuda")
    block = wide[:, 1]
    x, h = residual_norm(block, block, after="rms", before="layer")
    y, k = residual_norm(block.clone(), block.clone(), after="rms", before="layer")
    assert torch.equal(x, y) and torch.equal(h, k) and torch.isfinite(h).all()
    spoiled = block.clone()
    spoiled[7, 5], spoiled[9, 0] = float("nan"), float("inf")
    x, h = residual_norm(spoiled, spoiled, after="rms", before="layer")
    rest = [i for i in range(50) if i not in (7, 9)]
    assert torch.equal(x[rest], y[rest]) and torch.equal(h[rest], k[rest]) and x[7].isnan().all() and h[9].isnan().all()


def test_refusals_of_the_norms_on_the_gpu():
    x = torch.randn(4, 64, device="cuda")
    for args, options, match in (((x.half(),), {}, "float32 or bfloat16"), ((x, x[:3]), {}, "residual has shape"),
                                 ((x, x.cpu()), {}, "one device"), ((x, None, x[:, :32]), {}, "gate of shape"),
                                 ((x,), dict(after=("max",)), "must be None or"), ((x,), dict(after=("rms", x[0, :3])), "vectors of 64"),
                                 ((x,), dict(before=("rms", x[0].cpu())), "one device"), ((x,), dict(activation="relu"), "activation"),
                                 ((torch.zeros(2, 16385, device="cuda"),), {}, "1 to 16384"),
                                 ((torch.zeros(2, 0, device="cuda"),), {}, "1 to 16384")):
        with pytest.raises(RuntimeError, match=match):
            residual_norm(*args, **options)


@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
@pytest.mark.parametrize("dtype", [F, B])
def test_gates_far_out(activation, dtype):
    """Gates that close or open entirely: factors and slopes are what they tend to, also at the type's lowest value."""
    ends = [torch.finfo(dtype).min, -1e4, -200.0, -100.0, -95.0, -90.0, -89.0, -88.0, -87.0, -60.0, -20.0, 0.0, 20.0, 87.0, 89.0, 100.0,
            1e4]
    gen = torch.Generator().manual_seed(1)
    block = (1 + torch.rand(8, 64 * len(ends), generator=gen)).to(dtype)
    gate = (torch.tensor(ends).repeat_interleave(64)[None] * (1 + 0.004 * torch.rand(8, 64 * len(ends), generator=gen))).to(dtype)
    gate = gate.clamp_min(torch.finfo(dtype).min)
    b, g = block.cuda().requires_grad_(True), gate.cuda().requires_grad_(True)
    x, _ = residual_norm(b, gate=g, activation=activation)
    got = torch.autograd.grad(x, [b, g], torch.ones_like(x))
    wb, wg = block.double().requires_grad_(True), gate.double().requires_grad_(True)
    s = 1 / (1 + torch.exp(-wg.clamp_min(-700.0)))
    want = wb * (s if activation == "sigmoid" else wg.clamp_min(-700.0) * s)
    exact = torch.autograd.grad(want, [wb, wg], torch.ones_like(want))
    for a, e in zip((x, *got), (want, *exact)):
        a = a.detach().double().cpu()
        assert torch.isfinite(a).all()
        # (element by element: twelve half steps at most, 2^-24 each, of the factors and their products; and what is below 2^-118
        # may be zero: 88 x 2^-125)
        assert ((a - e.detach()).abs() <= (2.0 ** -20 + torch.finfo(dtype).eps / 2) * e.detach().abs() + 2.0 ** -118).all()
    ends = torch.tensor([[-float("inf"), float("inf"), float("nan")]], device="cuda", dtype=dtype).requires_grad_(True)
    x, _ = residual_norm(torch.ones(1, 3, device="cuda", dtype=dtype), gate=ends, activation=activation)
    (slope,) = torch.autograd.grad(x, ends, torch.ones_like(x))
    top = 1.0 if activation == "sigmoid" else float("inf")
    assert x[0, 0] == 0 and x[0, 1] == top and x[0, 2].isnan()
    assert slope[0, 0] == 0 and slope[0, 1] == (0 if activation == "sigmoid" else 1) and slope[0, 2].isnan()


@pytest.mark.parametrize("gate", [(5, 7, 64), (5, 1, 64), (1, 1, 64), (64,), (7, 64), (1, 7, 64), (5, 7, 1), (2, 7, 64), (3, 5, 7, 64)])
def test_plain_and_watched_calls_agree_on_gates(gate):
    """Gates of every broadcast, on rows with one and two strides, through both ways of a call."""
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(5, 7, 2 * 64, generator=gen).cuda()
    w = torch.rand(64, generator=gen).cuda().add_(0.5).requires_grad_(True)
    g = torch.randn(*gate, generator=gen).cuda().requires_grad_(True)
    bad = gate in ((5, 7, 1), (2, 7, 64), (3, 5, 7, 64))
    for block in (wide[..., 64:], wide[..., :64].contiguous(), wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :64]):
        block = block.detach().requires_grad_(True)
        call = lambda: residual_norm(block, block, g, after=("rms", w), before="layer", activation="silu")  # noqa: E731
        if bad:
            with pytest.raises(RuntimeError, match="gate of shape"):
                call()
            continue
        plain = call()
        go = [torch.ones_like(t) for t in plain]
        first = [*plain, *torch.autograd.grad(plain, [block, g, w], go)]
        with watched():
            seen = call()
        second = [*seen, *torch.autograd.grad(seen, [block, g, w], go)]
        with torch.no_grad():
            third = call()
        assert all(torch.equal(a, b) for a, b in zip(first, second)) and all(torch.equal(a, b) for a, b in zip(first, third))
        b, gg = (t.detach().double().cpu() for t in (block, g))
        want = norm.residual_norm(b, b, gg, ("rms", w.detach().double().cpu()), ("layer",), 1.0, "silu")
        assert norm.far(plain[0].detach(), want[0]) <= norm.FP32 and norm.far(plain[1].detach(), want[1]) <= norm.FP32


@pytest.mark.parametrize("width", [3, 5, 9, 15, 37, 101, 1023, 4093, 8195])
@pytest.mark.parametrize("dtype", [F, B])
def test_tails_of_rows_keep_to_themselves(width, dtype):
    """Rows that end inside a lane's eight values, with NaN before and behind them."""
    gen = torch.Generator().manual_seed(width)
    names = ("block", "residual", "gate")
    t = {n: torch.randn(9, width, generator=gen).to(dtype) for n in names}
    inside = {}
    for n in names:
        buffer = torch.full((9, width + 13), float("nan"), device="cuda", dtype=dtype)
        view = buffer[:, 7:7 + width]
        view.copy_(t[n])
        inside[n] = view
    go = [torch.ones(9, width, device="cuda", dtype=dtype)] * 2
    for a, b in zip(gradients(inside, "layer", "rms", go), gradients({n: x.cuda() for n, x in t.items()}, "layer", "rms", go)):
        assert torch.isfinite(a).all() and torch.equal(a, b)
