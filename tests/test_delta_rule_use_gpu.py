"""The gated delta rule as programs call it: strides and alignments, masked places, extreme decays and keys, streams,
captured graphs, watched calls, long offsets, and that nothing else is written."""
import pytest
import torch

import delta_reference as ref
from fast_transformers_amd.delta_rule import GatedDeltaRule, gated_delta_rule, gated_delta_step

pytestmark = pytest.mark.gpu


def results(args, go, gs, needed=None, **options):
    """[out, state, gradients] of a call and its backward."""
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = gated_delta_rule(*leaves, return_state=True, **options)
    return [out.detach(), state.detach(), *torch.autograd.grad([out, state], leaves, [go, gs])]


def wanted(args, go, gs, **options):
    wide = [t.detach().double().cpu().requires_grad_(True) for t in args]
    options.setdefault("scale", args[0].shape[3] ** -0.5)
    out, state = ref.rule(*wide, **options)
    return [out, state, *torch.autograd.grad([out, state], wide, [go.double().cpu(), gs.double().cpu()])]


def seeds(args, device="cuda"):
    gen = torch.Generator().manual_seed(77)
    go = torch.randn(args[2].shape, generator=gen).to(args[2].dtype)
    return go.to(device), (0.3 * torch.randn(args[5].shape, generator=gen)).to(device)


def check(got, want):
    errors = [ref.far(a, b) for a, b in zip(got, want)]
    print(["%.2g" % e for e in errors], flush=True)
    for a, e in zip(got, errors):
        assert e <= ref.tolerance(a.dtype), errors


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scalars", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype, scalars):
    args = ref.inputs(2, 4, 2, 100, 64, 32, dtype=dtype, scalars=scalars, device="cuda")
    go, gs = seeds(args)
    want = wanted(args, go, gs)
    check(results(args, go, gs), want)                                   # views of (N, L, H, X)
    check(results([t.contiguous() for t in args], go, gs), want)         # (N, H, L, X)

    def inside(t):  # rows of a wider buffer, off the 16-byte grid
        buffer = torch.full((*t.shape[:-1], t.shape[-1] + 7), float("nan"), device="cuda", dtype=t.dtype)
        view = buffer[..., 3:3 + t.shape[-1]]
        view.copy_(t)
        return view

    def apart(t):  # values that lie apart
        buffer = torch.full((*t.shape, 2), float("nan"), device="cuda", dtype=t.dtype)
        buffer[..., 0] = t
        return buffer[..., 0]
    for form in (inside, apart):
        moved = [form(t) for t in args]
        check(results(moved, form(go), form(gs)), want)
    turned = [t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim()))) for t in args]
    check(results(turned, go, gs), want)


def test_one_row_for_all_and_one_tensor_twice():
    args = ref.inputs(2, 3, 3, 70, 32, 48, device="cuda")
    go, gs = seeds(args)
    shared = [t[:1].expand_as(t) for t in args[:5]] + [args[5]]          # zero strides over the sequences
    got = results(shared, go, gs)
    check(got, wanted(shared, go, gs))
    q = args[0].detach().requires_grad_(True)
    out = gated_delta_rule(q, q, args[2], args[3], args[4])              # queries that are the keys
    (grad,) = torch.autograd.grad(out, q, go)
    wide = q.detach().double().cpu().requires_grad_(True)
    want, _ = ref.rule(wide, wide, *(t.double().cpu() for t in args[2:5]), scale=32 ** -0.5)
    assert ref.far(grad, torch.autograd.grad(want, wide, go.double().cpu())[0]) <= ref.FP32


@pytest.mark.parametrize("L", [5, 100])
def test_masked_places_may_hold_anything(L):
    for dtype in (torch.float32, torch.bfloat16):
        args = ref.inputs(3, 2, 1, L, 64, 32, dtype=dtype, device="cuda")
        go, gs = seeds(args)
        lengths = torch.tensor([L - 2, 0, 1], device="cuda")
        clean = results(args, go, gs, lengths=lengths)
        check(clean, wanted(args, go, gs, lengths=lengths.cpu()))
        dirty = [t.clone() for t in args]
        for t in dirty[:5]:
            t[0, :, L - 2:], t[1], t[2, :, 1:] = float("nan"), float("inf"), torch.finfo(t.dtype).min
        spoiled = go.clone()
        spoiled[0, :, L - 2:], spoiled[1] = float("nan"), float("inf")
        for a, b in zip(results(dirty, spoiled, gs, lengths=lengths), clean):
            assert torch.equal(a, b)
        for grad in clean[2:7]:
            assert not grad[1].any() and not grad[0, :, L - 2:].any() and not grad[2, :, 1:].any()


def test_lengths_out_of_range_are_the_ends():
    args = ref.inputs(2, 2, 2, 70, 16, 16, device="cuda")
    got = gated_delta_rule(*args, lengths=torch.tensor([1000, -3], device="cuda"), return_state=True)
    want = gated_delta_rule(*args, lengths=torch.tensor([70, 0], device="cuda"), return_state=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("L", [6, 140])
def test_extreme_decays_and_betas(L):
    args = ref.inputs(2, 2, 2, L, 64, 64, device="cuda", seed=4)
    g, b = args[3], args[4]
    g[0, 0, L // 2] = -float("inf")                                      # the state is forgotten
    g[0, 1] = 0.0                                                        # and never
    g[1, 0] = -30.0                                                      # sums beyond what exp can hold
    g[1, 1, ::3] = -torch.finfo(torch.float32).max
    b[0, 0, 1], b[1, 1] = 0.0, 1.0
    b[0, 1, ::2] = 0.0
    go, gs = seeds(args)
    got = results(args, go, gs)
    wide = [t.double().cpu() for t in args]
    # (the definition's own gradient at a decay of -inf or nothing: 0 x inf; what it decays to is zero either way)
    wide[3] = wide[3].clamp_min(-1000.0)
    check(got, wanted(wide, go, gs))


def test_keys_that_resemble_each_other():
    """Equal keys written with beta 1 and no decay: powers of their products would cancel; M is all ones."""
    N, H, L, E, M = 1, 2, 130, 64, 32
    args = ref.inputs(N, H, H, L, E, M, device="cuda", seed=6)
    args[1].copy_(args[1][:, :, :1].expand_as(args[1]))
    args[3].zero_()
    args[4].fill_(1.0)
    go, gs = seeds(args)
    check(results(args, go, gs), wanted(args, go, gs))


def test_offsets_beyond_32_bits():
    """Rows 2^22 elements apart: the last positions lie 5 GB behind the first."""
    L, step = 600, 1 << 22
    args = ref.inputs(1, 1, 1, L, 32, 32, dtype=torch.bfloat16, device="cuda")
    buffer = torch.zeros((L, step), device="cuda", dtype=torch.bfloat16)
    far = []
    for i, t in enumerate(args[:3]):
        view = buffer[:, 64 * i:64 * i + 32]
        view.copy_(t[0, 0])
        far.append(view[None, None])
    go, gs = seeds(args)
    for a, b in zip(results(far + args[3:], go, gs), results(args, go, gs)):
        assert torch.equal(a, b)


def test_state_is_a_view_and_nothing_else_is_written():
    q, k, v, g, b, s0 = ref.inputs(3, 2, 2, 1, 24, 20, device="cuda")
    for M in (20, 19):
        buffer = torch.full((4, 3, 2, 30, 32), 7.0, device="cuda")
        state = buffer[1, :, :, 3:27, 4:4 + M]
        state.copy_(s0[..., :M])
        gated_delta_step(q[:, :, 0], k[:, :, 0], v[:, :, 0, :M], g[:, :, 0], b[:, :, 0], state)
        want = ref.rule(*(t.double().cpu() for t in (q, k, v[..., :M], g, b, s0[..., :M])), scale=24 ** -0.5)[1]
        assert ref.far(state, want) <= ref.FP32
        inside = torch.zeros_like(buffer, dtype=torch.bool)
        inside[1, :, :, 3:27, 4:4 + M] = True
        assert (buffer[~inside] == 7.0).all()


def test_refusals_on_the_gpu():
    q, k, v, g, b, s0 = ref.inputs(2, 4, 2, 9, 16, 8, device="cuda")
    for bad, match in (((q, k[:, :, :4], v, g, b), "keys"), ((q, k, v.bfloat16(), g, b), "dtype"), ((q, k, v, g[:, :2], b), "log_decay"),
                       ((q, k, v, g, b.double()), "float32 or bfloat16"), ((q.half(), k.half(), v.half(), g, b), "float32 or bfloat16"),
                       ((q, k, v, g.cpu(), b), "device"), ((q[:, :1].expand(2, 3, 9, 16), k[:, :1].expand(2, 3, 9, 16), v, g, b), "multiple"),
                       ((q, k, v, g, b, s0[:, :, :, :3]), "initial_state"), ((q, k, v, g, b, s0.double()), "initial_state"),
                       ((torch.zeros(2, 2, 9, 129, device="cuda"),) * 2 + (v, g, b), "1 to 128"),
                       ((torch.zeros(2, 2, 9, 0, device="cuda"),) * 2 + (v, g, b), "1 to 128")):
        with pytest.raises(RuntimeError, match=match):
            gated_delta_rule(*bad)
    with pytest.raises(RuntimeError, match="lengths"):
        gated_delta_rule(q, k, v, g, b, lengths=torch.tensor([9], device="cuda"))
    one = [t[:, :, 0] for t in (q, k, v, g, b)]
    with pytest.raises(RuntimeError, match="contiguous"):
        gated_delta_step(*one, s0.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(RuntimeError, match="overlap"):
        gated_delta_step(*one, s0[:1].expand_as(s0))
    with pytest.raises(RuntimeError, match="state"):
        gated_delta_step(*one, s0.cpu())
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        gated_delta_step(*one, s0.clone().requires_grad_(True))


def test_watched_calls_take_the_python_function():
    args = ref.inputs(2, 2, 1, 80, 32, 32, device="cuda")
    go, gs = seeds(args)
    plain = results(args, go, gs)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t, lambda t: t):
        watched = results(args, go, gs)
    assert packed and all(torch.equal(a, b) for a, b in zip(plain, watched))
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = GatedDeltaRule.apply(*leaves, None, 32 ** -0.5, False)
    assert torch.equal(out, plain[0]) and torch.equal(state, plain[1])


def test_some_gradients_and_one_graph_twice():
    args = ref.inputs(2, 4, 2, 90, 64, 32, device="cuda")
    go, gs = seeds(args)
    every = results(args, go, gs)
    for i in range(6):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate(args)]
        out, state = gated_delta_rule(*leaves, return_state=True)
        for _ in range(2):
            (grad,) = torch.autograd.grad([out, state], [leaves[i]], [go, gs], retain_graph=True)
            assert torch.equal(grad, every[2 + i])
    # the state alone, the outputs alone
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = gated_delta_rule(*leaves, return_state=True)
    zero = results(args, torch.zeros_like(go), gs)
    got = torch.autograd.grad(state, leaves, gs, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, zero[2:]))
    zero = results(args, go, torch.zeros_like(gs))
    got = torch.autograd.grad(out, leaves, go)
    assert all(torch.equal(a, b) for a, b in zip(got, zero[2:]))


def test_differences():
    """Gradients against central differences of the outputs, in directions of every input."""
    args = ref.inputs(1, 2, 1, 70, 16, 8, device="cuda", seed=9)
    go, gs = seeds(args)
    grads = results(args, go, gs, normalize=True)[2:]
    gen = torch.Generator(device="cuda").manual_seed(3)

    def loss(moved):
        out, state = gated_delta_rule(*moved, normalize=True, return_state=True)
        return (out.double() * go).sum() + (state.double() * gs).sum()
    for i, (t, grad) in enumerate(zip(args, grads)):
        d = torch.randn(t.shape, generator=gen, device="cuda")
        d = d / d.norm()
        h = 2.0 ** -6
        up, down = ([x + s * h * d if j == i else x for j, x in enumerate(args)] for s in (1, -1))
        slope = ((loss(up) - loss(down)) / (2 * h)).item()
        # a difference's error: rounding of two losses (terms of size |go| |out|, 2^-24 of them each, over 2 h) and the third
        # derivative's h^2 / 6 times a slope's size
        size = (go.norm() * 1.0 + gs.norm()).item()
        assert abs(slope - (grad.double() * d).sum().item()) <= size * (2.0 ** -23 / h * 8 + h * h), (i, slope)


def test_other_streams_and_two_calls_at_once():
    args = ref.inputs(4, 8, 8, 500, 64, 64, dtype=torch.bfloat16, device="cuda")
    other = ref.inputs(4, 8, 8, 500, 64, 64, dtype=torch.bfloat16, device="cuda", seed=5)
    go, gs = seeds(args)
    want = [results(a, go, gs) for a in (args, other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, (s, a) in enumerate(zip(streams, (args, other))):
            with torch.cuda.stream(s):
                got[i] = results(a, go, gs)
        torch.cuda.synchronize()
        for x, y in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_captured_training_steps():
    """Two graphs of forward and backward, replayed in turn and with eager work between, give what eager calls give."""
    cases = []
    for seed in (1, 2):
        args = ref.inputs(2, 4, 2, 200, 64, 64, dtype=torch.bfloat16, device="cuda", seed=seed)
        cases.append((args, *seeds(args)))
    inputs = [[t.detach().clone().requires_grad_(True) for t in a] for a, _, _ in cases]
    graphs, outs = [], []
    for leaves, (_, go, gs) in zip(inputs, cases):
        def once():
            out, state = gated_delta_rule(*leaves, normalize=True, return_state=True)
            return [out, state, *torch.autograd.grad([out, state], leaves, [go, gs])]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                once()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([t.detach() for t in once()])
        graphs.append(graph)
    for turn in range(4):
        new = [ref.inputs(2, 4, 2, 200, 64, 64, dtype=torch.bfloat16, device="cuda", seed=10 + 2 * turn + i) for i in range(2)]
        for leaves, values in zip(inputs, new):
            with torch.no_grad():
                for leaf, t in zip(leaves, values):
                    leaf.copy_(t)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for values, out, (_, go, gs) in zip(new, outs, cases):
            for a, b in zip(results(values, go, gs, normalize=True), out):
                assert torch.equal(a, b), turn


def test_results_are_the_same_every_time():
    args = ref.inputs(3, 8, 2, 333, 128, 96, dtype=torch.bfloat16, device="cuda")
    go, gs = seeds(args)
    first = results(args, go, gs, normalize=True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, results(args, go, gs, normalize=True)))


def test_pieces_of_a_sequence_carry_the_state():
    args = ref.inputs(2, 4, 4, 300, 64, 64, dtype=torch.bfloat16, device="cuda")
    whole, last = gated_delta_rule(*args, return_state=True)
    state, outs = args[5], []
    for lo, hi in ((0, 1), (1, 8), (8, 100), (100, 164), (164, 292), (292, 300)):
        out, state = gated_delta_rule(*(t[:, :, lo:hi] for t in args[:5]), state, return_state=True)
        outs.append(out)
    assert ref.far(state, last) <= ref.FP32
    assert ref.far(torch.cat(outs, 2), whole) <= 2 * ref.BF16


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [1, 2, 4, 5, 66, 130])
@pytest.mark.parametrize("strength", [None, -2.0, -4.0, -12.0])
def test_gradients_of_few_or_strong_decays(dtype, L, strength):
    """They are small beside what the positions pass to and fro: found from what crosses a position, not as a difference."""
    for E, M, state in ((64, 64, True), (100, 80, False), (37, 51, True)):
        args = ref.inputs(2, 4, 2, L, E, M, dtype=dtype, device="cuda", seed=L)
        if strength is not None:
            args[3].copy_(strength - args[3].abs())
        if not state:
            args[5].zero_()
        go, gs = seeds(args)
        got, want = results(args, go, gs, normalize=True), wanted(args, go, gs, normalize=True)
        check(got, want)
        if not state:  # nothing decays at the first position
            leaves = [t.detach().requires_grad_(True) for t in args[:5]]
            o, s = gated_delta_rule(*leaves, normalize=True, return_state=True)
            (dg,) = torch.autograd.grad([o, s], [leaves[3]], [go, gs])
            if L <= 4 or strength is not None:
                assert not dg[:, :, 0].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N, H, Hk, L, E, M", [(1, 2, 1, 1000, 64, 64), (3, 1, 1, 1100, 37, 21), (2, 2, 2, 1290, 128, 128), (2, 1, 1, 800, 70, 130),
                                               (1, 1, 1, 3100, 16, 16)])
def test_few_long_chains_are_walked_in_segments(dtype, N, H, Hk, L, E, M):
    args = ref.inputs(N, H, Hk, L, E, M, dtype=dtype, device="cuda", seed=L)
    args[3][:, :1].mul_(0.02)                                            # (a head that remembers over segments)
    go, gs = seeds(args)
    for lengths in (None, [L] + [L // 2, 5][:N - 1]):
        got = results(args, go, gs, normalize=True, lengths=None if lengths is None else torch.tensor(lengths, device="cuda"))
        want = wanted(args, go, gs, normalize=True, lengths=None if lengths is None else torch.tensor(lengths))
        check(got, want)
        out, state = gated_delta_rule(*args, normalize=True, return_state=True,
                                      lengths=None if lengths is None else torch.tensor(lengths, device="cuda"))
        assert torch.equal(out, got[0]) and torch.equal(state, got[1])
    zero = args[:5] + [torch.zeros_like(args[5])]
    out, state = gated_delta_rule(*args[:5], return_state=True)          # without a state
    again, last = gated_delta_rule(*zero, return_state=True)
    assert torch.equal(out, again) and torch.equal(state, last)


@pytest.mark.parametrize("seed", range(12))
def test_drawn_shapes(seed):
    """Sizes, heads, lengths, layouts and options as they come, on every route of the kernels."""
    import random
    rng = random.Random(seed)
    Hk = rng.choice([1, 2, 3])
    N, H, L = rng.choice([1, 2, 5]), Hk * rng.choice([1, 2, 3]), rng.choice([1, 7, 9, 63, 64, 65, 200, 777, 1300])
    E, M = rng.choice([1, 3, 16, 33, 64, 65, 96, 128]), rng.choice([1, 5, 16, 48, 64, 100, 128, 512])
    dtype = rng.choice([torch.float32, torch.bfloat16])
    if M == 512:
        N, H, Hk = 1, 2, 1
    normalize = E > 3 and rng.random() < 0.5      # (the gradient of a row's direction is all cancellation where it has one value)
    args = ref.inputs(N, H, Hk, L, E, M, dtype=dtype, scalars=rng.choice([torch.float32, dtype]), device="cuda", seed=seed)
    if rng.random() < 0.5:
        args = [t.contiguous() for t in args]
    go, gs = seeds(args)
    lengths = rng.choice([None, [rng.randint(0, L) for _ in range(N)]])
    print(N, H, Hk, L, E, M, dtype, normalize, lengths, flush=True)
    got = results(args, go, gs, normalize=normalize, lengths=None if lengths is None else torch.tensor(lengths, device="cuda"))
    check(got, wanted(args, go, gs, normalize=normalize, lengths=None if lengths is None else torch.tensor(lengths)))
