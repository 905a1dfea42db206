"""The operators of gated delta-rule language models: the rule over whole sequences, its single step, and the
norms around a block, each in its plain form and as the framework's call.

The rule, per chain of a value head, on a state S of E x M (k, q of E values, v of M):

    S' = exp(g_t) S_{t-1},  z_t = v_t - S'^T k_t,  S_t = S' + k_t (beta_t z_t)^T,  o_t = S_t^T q_t

with ``H`` value heads on ``Hk`` key heads, q scaled by E^-1/2, both optionally brought to length one
(``normalize``), and positions at or past a sequence's length left out (``ragged``).

The norms around a block, per row:

    x = residual + scale act(gate) norm_after(block),   h = norm_before(x)

Cases are dicts of plain values.  ``kind``: "prefill" (the rule in inference, state in and out), "train" (the
rule, forward and backward), "step" (one token, state in place), "norm" and "norm_train".
"""
import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_CHUNK = 64
_EPS = 1e-6


def _rule(kind, N, H, Hk, L, E, M, dtype, ragged=False, normalize=True):
    return dict(kind=kind, N=N, H=H, Hk=Hk, L=L, E=E, M=M, dtype=dtype, ragged=ragged, normalize=normalize)


def _step(N, H, Hk, E, M, dtype, normalize=True):
    return dict(kind="step", N=N, H=H, Hk=Hk, E=E, M=M, dtype=dtype, normalize=normalize)


def _norm(kind, N, L, D, dtype, stream, after, before, gate, activation, scale=1.0):
    return dict(kind=kind, N=N, L=L, D=D, dtype=dtype, stream=stream, after=after, before=before, gate=gate,
                activation=activation, scale=scale)


def listed():
    return [
        # one token of one sequence being generated: launch and latency only
        dict(_step(1, 8, 8, 64, 64, "fp32"), name="step_one_sequence"),
        # one token for each of 256 sequences, two value heads on every key head: the states' traffic
        dict(_step(256, 16, 8, 128, 128, "bf16"), name="step_many_sequences"),
        # the next 2048 tokens of four half-precision prompts, state handed in and out
        dict(_rule("prefill", 4, 16, 16, 2048, 128, 128, "bf16"), name="prefill_bf16"),
        # a padded batch of short prompts with odd head widths and lengths that divide nothing
        dict(_rule("prefill", 9, 11, 11, 331, 25, 33, "fp32", ragged=True, normalize=False), name="prefill_odd_ragged"),
        # the training step at the size of the linear attention's quick start
        dict(_rule("train", 10, 8, 8, 1000, 64, 64, "fp32"), name="train_quickstart"),
        # the training step of a layer of wide heads, two value heads on every key head
        dict(_rule("train", 8, 16, 8, 4096, 128, 128, "bf16"), name="train_wide_bf16"),
        # one long sequence: few chains, many chunks one after the other
        dict(_rule("train", 1, 16, 16, 16384, 64, 64, "bf16"), name="train_long_bf16"),
        # the norms between two blocks for one token of 32 sequences
        dict(_norm("norm", 32, 1, 512, "bf16", "bf16", "rms", "rms", "none", "none"), name="norm_step"),
        # the encoder's width, fp32, layer norms, a gate and a scale of every sequence's own: training
        dict(_norm("norm_train", 10, 4096, 512, "fp32", "fp32", "layer", "layer", "sequence", "none", 0.5),
             name="norm_train_fp32"),
        # a wide model's stream kept in fp32 beside half-precision blocks, gated by every token: training
        dict(_norm("norm_train", 4, 4096, 4096, "bf16", "fp32", "rms", "rms", "full", "sigmoid"),
             name="norm_train_wide_mixed"),
        # the gated norm of the rule's outputs: rows of one head each, no residual: training
        dict(_norm("norm_train", 8, 65536, 128, "bf16", "none", "rms", "none", "full", "silu"),
             name="norm_train_heads"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm, odd as often as not."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["prefill", "train", "step", "norm", "norm_train"])
    while True:
        if kind in ("norm", "norm_train"):
            stream = rng.choice(["none", "fp32", "bf16"])
            gate = rng.choice(["none", "full", "sequence", "channel"])
            before = rng.choice(["none", "rms", "layer"])
            after = rng.choice(["none", "rms", "layer"])
            case = _norm(kind, _spread(rng, 1, 64), _spread(rng, 1, 8192), _spread(rng, 32, 8192),
                         rng.choice(["fp32", "bf16"]), stream, after if before != "none" or after != "none" else "rms",
                         before, gate, rng.choice(["none", "sigmoid", "silu"]) if gate != "none" else "none",
                         rng.choice([1.0, 0.5]))
        else:
            Hk = _spread(rng, 1, 16)
            H = Hk * rng.choice([1, 1, 2, 4])
            E, M = (rng.choice([32, 64, 96, 128, _spread(rng, 8, 128)]) for _ in range(2))
            dtype, normalize = rng.choice(["fp32", "bf16"]), rng.choice([True, False])
            if kind == "step":
                case = _step(_spread(rng, 1, 256), H, Hk, E, M, dtype, normalize)
            else:
                case = _rule(kind, _spread(rng, 1, 16), H, Hk, _spread(rng, 1, 8192), E, M, dtype,
                             rng.choice([True, False]), normalize)
        w = work(case)
        if w["bytes"] <= 1.2e9 and w["flops"] <= 1.8e11:
            return case


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _decays(gen, *shape):
    """Log decays as such models make them: -exp(a) softplus(x), from a hundredth to a few."""
    rates = torch.exp(-4 + 4 * torch.rand(shape[1], generator=gen, device="cuda"))
    return -rates.view(1, -1, *[1] * (len(shape) - 2)) * torch.nn.functional.softplus(_randn(gen, *shape))


def _inputs_rule(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    N, H, Hk, E, M = (case[x] for x in ("N", "H", "Hk", "E", "M"))
    row = () if case["kind"] == "step" else (case["L"],)
    # projections lie as (N, L, heads, width) and are handed over as views
    turn = (lambda t: t) if case["kind"] == "step" else (lambda t: t.permute(0, 2, 1, 3))
    q, k = (turn(_randn(gen, N, *row, Hk, E).to(dtype)) for _ in range(2))
    if not case["normalize"]:
        q, k = (torch.nn.functional.normalize(t.float(), dim=-1).to(dtype) for t in (q, k))
    v = turn(_randn(gen, N, *row, H, M).to(dtype))
    state = dict(q=q, k=k, v=v, g=_decays(gen, N, H, *row), b=torch.sigmoid(_randn(gen, N, H, *row)),
                 s0=_randn(gen, N, H, E, M) * 0.3, scale=E ** -0.5, normalize=case["normalize"], lengths=None)
    if case.get("ragged"):
        lengths = torch.randint(0, case["L"] + 1, (N,), generator=gen, device="cuda")
        lengths[0] = case["L"]
        state["lengths"] = lengths
    if case["kind"] == "train":
        state["go"] = _randn(gen, N, H, case["L"], M).to(dtype)
        state["s0"] = None
    return state


_RULE_LEAVES = ("q", "k", "v", "g", "b")
_NORM_LEAVES = ("block", "residual", "gate", "aw", "ab", "bw", "bb")


def _inputs_norm(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    N, L, D = case["N"], case["L"], case["D"]
    shapes = {"full": (N, L, D), "sequence": (N, 1, D), "channel": (D,)}
    s = dict(block=(1 + _randn(gen, N, L, D)).to(dtype), residual=None, gate=None, aw=None, ab=None, bw=None, bb=None)
    if case["stream"] != "none":
        s["residual"] = (2 * _randn(gen, N, L, D)).to(_DTYPES[case["stream"]])
    if case["gate"] != "none":
        s["gate"] = _randn(gen, *shapes[case["gate"]]).to(dtype)
    for name, x in (("after", "a"), ("before", "b")):
        if case[name] != "none":
            s[x + "w"] = 1 + 0.1 * _randn(gen, D)
        if case[name] == "layer":
            s[x + "b"] = 0.1 * _randn(gen, D)
    if case["kind"] == "norm_train":
        s["gx"] = _randn(gen, N, L, D).to(s["residual"].dtype if s["residual"] is not None else dtype)
        s["gh"] = _randn(gen, N, L, D).to(dtype) if case["before"] != "none" else None
    return s


def prepare(case, seed):
    if case["kind"] in ("norm", "norm_train"):
        state, leaves = _inputs_norm(case, seed), _NORM_LEAVES
    else:
        state, leaves = _inputs_rule(case, seed), _RULE_LEAVES
    if case["kind"] in ("train", "norm_train"):
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_(True)
    state["case"] = case
    return state


# ---- the plain forms ----

def _unit(x, normalize):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + _EPS) if normalize else x


def _plain_rule(q, k, v, g, b, s0, scale, normalize, lengths):
    """The rule in chunks of 64 positions, in fp32: everything inside the chunks at once, then the states one
    chunk after the other (the recurrence leaves no other way)."""
    N, H, L, M = v.shape
    E, group, dtype = q.shape[3], H // q.shape[1], v.dtype
    q, k = (_unit(t.float(), normalize).repeat_interleave(group, 1) for t in (q, k))
    q, v, g, b = q * scale, v.float(), g.float(), b.float()
    if lengths is not None:
        valid = (torch.arange(L, device=q.device) < lengths[:, None])[:, None]
        q, k, v = (torch.where(valid[..., None], t, 0.0) for t in (q, k, v))
        g, b = (torch.where(valid, t, 0.0) for t in (g, b))
    pad = -L % _CHUNK
    C = (L + pad) // _CHUNK
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).reshape(N, H, C, _CHUNK, -1) for t in (q, k, v))
    g, b = (torch.nn.functional.pad(t, (0, pad)).reshape(N, H, C, _CHUNK) for t in (g, b))
    G = g.double().cumsum(-1)                                    # (differences of long sums)
    ones = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device)
    lower, strict = torch.tril(ones), torch.tril(ones, -1)
    D = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~lower, 0.0).float())
    rise, fall, last = G.exp().float(), (G[..., -1:] - G).exp().float(), G[..., -1].exp().float()
    kt = k.transpose(-1, -2)
    A = ((q @ kt) * D).masked_fill(~lower, 0.0)
    T = _inverse(((k @ kt) * D * b[..., None, :]).masked_fill(~strict, 0.0))
    own_part, state_part = T @ v, T @ (rise[..., None] * k)      # Z = own_part - state_part S
    write = (k * (b * fall)[..., None]).transpose(-1, -2)
    S = torch.zeros(N, H, E, M, device=q.device) if s0 is None else s0.float()
    states, errors = [], []
    for c in range(C):
        z = own_part[:, :, c] - state_part[:, :, c] @ S
        states.append(S)
        errors.append(z)
        S = last[:, :, c, None, None] * S + write[:, :, c] @ z
    out = (rise[..., None] * q) @ torch.stack(states, 2) + A @ (b[..., None] * torch.stack(errors, 2))
    return out.reshape(N, H, L + pad, M)[:, :, :L].to(dtype), S


def _inverse(strict):
    """(I + strict)^-1 of strictly lower triangular matrices of 64 x 64, from blocks of two, four, ... rows."""
    n = strict.shape[-1]
    inv = torch.eye(n, device=strict.device).expand_as(strict)
    index = torch.arange(n, device=strict.device)
    for bits in range(n.bit_length() - 1):
        block = index >> bits
        below = (block[:, None] == block[None, :] + 1) & (block[:, None] % 2 == 1)
        inv = inv - inv @ strict.masked_fill(~below, 0.0) @ inv
    return inv


def _plain_step(q, k, v, g, b, state, scale, normalize):
    group = v.shape[1] // q.shape[1]
    dtype = v.dtype
    q, k = (_unit(t.float(), normalize).repeat_interleave(group, 1) for t in (q, k))
    S = state * torch.exp(g.float())[..., None, None]
    z = v.float() - (S * k[..., None]).sum(2)
    S = S + k[..., None] * (b.float()[..., None] * z)[..., None, :]
    state.copy_(S)
    return (S * (scale * q)[..., None]).sum(2).to(dtype)


def _plain_norm_rows(x, kind, weight, bias):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
    return x if bias is None else x + bias


def _plain_norm(s, case):
    y = _plain_norm_rows(s["block"].float(), case["after"], s["aw"], s["ab"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        if case["activation"] != "none":
            sigmoid = 1 / (1 + torch.exp(-gate))
            gate = sigmoid if case["activation"] == "sigmoid" else gate * sigmoid
        y = gate * y
    x = case["scale"] * y
    if s["residual"] is not None:
        x = s["residual"].float() + x
    h = None
    if case["before"] != "none":
        h = _plain_norm_rows(x, case["before"], s["bw"], s["bb"]).to(s["block"].dtype)
    return x.to(s["block"].dtype if s["residual"] is None else s["residual"].dtype), h


# ---- one pass ----

@functools.lru_cache
def _package():
    root = os.path.abspath("fast-transformers_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from fast_transformers_amd import delta_rule, norms
    return delta_rule, norms


def _gradients(outs, grads, s, leaves):
    names = [n for n in leaves if s[n] is not None]
    pairs = [(o, g) for o, g in zip(outs, grads) if o is not None and g is not None]
    got = torch.autograd.grad([o for o, _ in pairs], [s[n] for n in names], [g for _, g in pairs])
    return {"grad_" + n: t for n, t in zip(names, got)}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        if own:
            spec = lambda name, w, b: None if name == "none" else (name, w) if b is None else (name, w, b)  # noqa: E731
            x, h = _package()[1].residual_norm(
                s["block"], s["residual"], s["gate"], after=spec(case["after"], s["aw"], s["ab"]),
                before=spec(case["before"], s["bw"], s["bb"]), scale=case["scale"],
                activation=None if case["activation"] == "none" else case["activation"], eps=_EPS)
        else:
            x, h = _plain_norm(s, case)
        outs = {"x": x} if h is None else {"x": x, "h": h}
        if kind == "norm":
            return outs
        return {**{n: t.detach() for n, t in outs.items()}, **_gradients((x, h), (s["gx"], s["gh"]), s, _NORM_LEAVES)}
    if kind == "step":
        args = (s["q"], s["k"], s["v"], s["g"], s["b"], s["s0"])
        if own:
            out = _package()[0].gated_delta_step(*args, scale=s["scale"], normalize=s["normalize"])
        else:
            out = _plain_step(*args, s["scale"], s["normalize"])
        return {"out": out, "state": s["s0"]}
    args = (s["q"], s["k"], s["v"], s["g"], s["b"], s["s0"])
    if own:
        out, state = _package()[0].gated_delta_rule(*args, scale=s["scale"], normalize=s["normalize"],
                                                    lengths=s["lengths"], return_state=True)
    else:
        out, state = _plain_rule(*args, s["scale"], s["normalize"], s["lengths"])
    if kind == "prefill":
        return {"out": out, "state": state}
    return {"out": out.detach(), "state": state.detach(), **_gradients((out,), (s["go"],), s, _RULE_LEAVES)}


def work(case):
    size = {"fp32": 4, "bf16": 2}
    b = size[case["dtype"]]
    if case["kind"] in ("norm", "norm_train"):
        rows = case["N"] * case["L"]
        stream = b if case["stream"] == "none" else size[case["stream"]]
        gate_rows = {"none": 0, "full": rows, "sequence": case["N"], "channel": 1}[case["gate"]]
        residual = 0 if case["stream"] == "none" else stream
        h = 0 if case["before"] == "none" else b
        # block, residual and gate in, x and h out
        row = case["D"] * (b + residual + stream + h)
        gate, params = gate_rows * case["D"] * b, 4 * case["D"] * (
            sum({"none": 0, "rms": 1, "layer": 2}[case[n]] for n in ("after", "before")))
        flops = 15.0 * rows * case["D"]
        if case["kind"] == "norm":
            return {"bytes": float(rows * row + gate + params), "flops": flops}
        # ... and the gradients of x and h in, those of block, residual, gate and parameters out
        more = case["D"] * (stream + h + b + residual)
        return {"bytes": float(rows * (row + more) + 2 * (gate + params)), "flops": 3 * flops}
    N, H, Hk, E, M = (case[x] for x in ("N", "H", "Hk", "E", "M"))
    L = case.get("L", 1)
    rows = N * L * (2 * Hk * E * b + 2 * H * M * b + 8 * H)
    flops = 7.0 * N * H * L * E * M  # S'^T k, the rank-one write, S^T q, the decay
    if case["kind"] == "train":
        # the state out; dO in and the gradients of q, k, v, g and beta out
        more = N * L * (2 * Hk * E * b + 2 * H * M * b + 8 * H)
        return {"bytes": float(rows + more + 4 * N * H * E * M), "flops": 3 * flops}
    return {"bytes": float(rows + 8 * N * H * E * M), "flops": flops}


# ---- the definition, in 64 bits ----

def _exact_rule(case, s):
    """One position after the other, forward, and backward with the states made again from every 64th."""
    kind, L = case["kind"], case["L"]
    N, H, E, M = (case[x] for x in ("N", "H", "E", "M"))
    group = H // case["Hk"]
    wide = lambda t: t.detach().double().repeat_interleave(group, 1).permute(2, 0, 1, 3).contiguous()  # noqa: E731
    q_raw, k_raw = wide(s["q"]), wide(s["k"])
    length = lambda t: (t.pow(2).sum(-1, keepdim=True) + _EPS).sqrt() if case["normalize"] else torch.ones_like(t[..., :1])  # noqa: E731
    nq, nk = length(q_raw), length(k_raw)
    q, k = q_raw / nq, k_raw / nk
    v = s["v"].detach().double().permute(2, 0, 1, 3).contiguous()
    g, b = (s[n].detach().double().permute(2, 0, 1).contiguous() for n in ("g", "b"))
    a = g.exp()
    live = torch.ones(L, N, 1, dtype=torch.float64, device=v.device)
    if s["lengths"] is not None:
        live = (torch.arange(L, device=v.device)[:, None] < s["lengths"]).double()[..., None]
        a, b = torch.where(live > 0, a, 1.0), b * live
    S = torch.zeros(N, H, E, M, dtype=torch.float64, device=v.device) if s["s0"] is None else s["s0"].double()
    scale, o = s["scale"], torch.empty_like(v)

    def forward(S, t):
        faded = a[t][..., None, None] * S
        z = v[t] - (k[t][..., None, :] @ faded)[..., 0, :]
        return faded, z, faded + k[t][..., :, None] * (b[t][..., None] * z)[..., None, :]

    kept = {}
    for t in range(L):
        if t % 64 == 0:
            kept[t] = S
        S = forward(S, t)[2]
        o[t] = live[t][..., None] * scale * (q[t][..., None, :] @ S)[..., 0, :]
    out = o.permute(1, 2, 0, 3)
    if kind == "prefill":
        return {"out": out, "state": S}
    go = s["go"].double().permute(2, 0, 1, 3).contiguous() * live[..., None] * scale
    dq, dk, dv, dg, db = (torch.empty_like(t) for t in (q, k, v, g, b))
    dS = torch.zeros_like(S)
    for start in sorted(kept, reverse=True):
        states, faded, zs = [kept[start]], [], []
        for t in range(start, min(L, start + 64)):
            f, z, after = forward(states[-1], t)
            states.append(after)
            faded.append(f)
            zs.append(z)
        for t in range(min(L, start + 64) - 1, start - 1, -1):
            f, z, after = faded[t - start], zs[t - start], states[t - start + 1]
            dq[t] = (after @ go[t][..., None])[..., 0]
            dS = dS + q[t][..., :, None] * go[t][..., None, :]
            du = (k[t][..., None, :] @ dS)[..., 0, :]
            dz = b[t][..., None] * du
            db[t] = (du * z).sum(-1)
            dv[t] = dz
            dk[t] = (dS @ (b[t][..., None] * z)[..., None])[..., 0] - (f @ dz[..., None])[..., 0]
            dS = dS - k[t][..., :, None] * dz[..., None, :]
            dg[t] = (dS * f).sum((-1, -2))
            dS = a[t][..., None, None] * dS
    if case["normalize"]:
        dq, dk = ((d - y * (y * d).sum(-1, keepdim=True)) / n for d, y, n in ((dq, q, nq), (dk, k, nk)))
    # (scale went into the gradient of the outputs above)
    back = lambda t: t.permute(1, 2, 0, 3)  # noqa: E731
    heads = lambda t: back(t * live[..., None]).reshape(N, case["Hk"], group, L, E).sum(2)  # noqa: E731
    return {"out": out, "state": S, "grad_q": heads(dq), "grad_k": heads(dk), "grad_v": back(dv * live[..., None]),
            "grad_g": (dg * live).permute(1, 2, 0), "grad_b": (db * live).permute(1, 2, 0)}


def _exact_step(case, s):
    group = case["H"] // case["Hk"]
    q, k = (s[n].double() for n in ("q", "k"))
    if case["normalize"]:
        q, k = (t / (t.pow(2).sum(-1, keepdim=True) + _EPS).sqrt() for t in (q, k))
    q, k = (t.repeat_interleave(group, 1)[..., None, :] for t in (q, k))
    faded = s["s0"].double() * s["g"].double().exp()[..., None, None]
    z = s["v"].double()[..., None, :] - k @ faded
    state = faded + k.transpose(-1, -2) @ (s["b"].double()[..., None, None] * z)
    return {"out": s["scale"] * (q @ state)[..., 0, :], "state": state}


def _exact_norm(case, s):
    wide = {n: None if s[n] is None else s[n].detach().double().requires_grad_(True) for n in _NORM_LEAVES}
    D = case["D"]

    def rows(x, kind, w, b):
        if kind == "none":
            return x
        if kind == "rms":
            return x / ((x.pow(2).sum(-1, keepdim=True) / D + _EPS).sqrt()) * w
        return (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + _EPS).sqrt() * w + b
    y = rows(wide["block"], case["after"], wide["aw"], wide["ab"])
    if s["gate"] is not None:
        y = y * {"none": lambda t: t, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[case["activation"]](wide["gate"])
    x = y * case["scale"] + (0 if s["residual"] is None else wide["residual"])
    h = None if case["before"] == "none" else rows(x, case["before"], wide["bw"], wide["bb"])
    outs = {"x": x} if h is None else {"x": x, "h": h}
    if case["kind"] == "norm":
        return {n: t.detach() for n, t in outs.items()}
    grads = [None if t is None else t.double() for t in (s["gx"], s["gh"])]
    return {**{n: t.detach() for n, t in outs.items()}, **_gradients((x, h), grads, wide, _NORM_LEAVES)}


def exact(case, seed):
    if case["kind"] in ("norm", "norm_train"):
        return _exact_norm(case, _inputs_norm(case, seed))
    s = _inputs_rule(case, seed)
    return _exact_step(case, s) if case["kind"] == "step" else _exact_rule(case, s)
