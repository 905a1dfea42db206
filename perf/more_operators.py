"""The operators of a model of decayed linear attention that is trained with dropout: the attention over whole
sequences, its single step, and the dropout behind a block, each in its plain form and as the framework's call.

The attention, per chain of a value head, on a state S of E x M (k, q of E values, v of M):

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t

with ``H`` value heads on ``Hk`` key heads, log decays g of every position or one for each head, and positions at or
past a sequence's length left out (``ragged``).

The dropout behind a block, per value i (counted over the block's rows, one after the other):

    x_i = residual_i + keep_i act(block_i + bias) / (1 - p),   keep_i = word_i >= p 2^32

where word_i is the word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) with the seed as its key and
(i // 4, offset) as its counter, 64 bits each.

Cases are dicts of plain values.  ``kind``: "prefill" (the attention in inference, state in and out), "train" (forward
and backward; with ``carry`` a state comes in and its gradient goes out), "step" (one token, state in place),
"dropout" and "dropout_train".
"""
import functools
import math
import os
import sys

import numpy
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_CHUNK = 64


def _rule(kind, N, H, Hk, L, E, M, dtype, decay, ragged=False, carry=False):
    return dict(kind=kind, N=N, H=H, Hk=Hk, L=L, E=E, M=M, dtype=dtype, decay=decay, ragged=ragged, carry=carry)


def _step(N, H, Hk, E, M, dtype, decay):
    return dict(kind="step", N=N, H=H, Hk=Hk, E=E, M=M, dtype=dtype, decay=decay)


def _dropout(kind, N, L, D, dtype, stream, bias, activation, p):
    return dict(kind=kind, N=N, L=L, D=D, dtype=dtype, stream=stream, bias=bias, activation=activation, p=p)


def listed():
    return [
        # one token of one sequence being generated: launch and latency only
        dict(_step(1, 8, 8, 64, 64, "fp32", "head"), name="step_one_sequence"),
        # one token for each of 256 sequences, two value heads on every key head: the states' traffic
        dict(_step(256, 16, 8, 128, 128, "bf16", "position"), name="step_many_sequences"),
        # the next 2048 tokens of four half-precision prompts, one decay for each head, state handed in and out
        dict(_rule("prefill", 4, 16, 16, 2048, 128, 128, "bf16", "head"), name="prefill_bf16"),
        # a padded batch of short prompts with odd head widths and lengths that divide nothing
        dict(_rule("prefill", 9, 11, 11, 331, 25, 33, "fp32", "position", ragged=True), name="prefill_odd_ragged"),
        # the training step at the size of the linear attention's quick start
        dict(_rule("train", 10, 8, 8, 1000, 64, 64, "fp32", "head"), name="train_quickstart"),
        # the training step of a layer of wide heads, two value heads on every key head
        dict(_rule("train", 8, 16, 8, 4096, 128, 128, "bf16", "position"), name="train_wide_bf16"),
        # one long sequence in pieces: few chains, many chunks one after the other, the state from the piece before
        dict(_rule("train", 1, 16, 16, 16384, 64, 64, "bf16", "position", carry=True), name="train_long_bf16"),
        # a few positions of a small batch: launches
        dict(_rule("train", 2, 4, 4, 17, 32, 32, "bf16", "position"), name="train_short"),
        # behind a block, onto the stream, for one short sequence: launch and latency only
        dict(_dropout("dropout", 1, 64, 512, "bf16", "bf16", False, "none", 0.1), name="dropout_short"),
        # behind a block of the encoder's width, onto the stream, in fp32: training
        dict(_dropout("dropout_train", 10, 4096, 512, "fp32", "fp32", False, "none", 0.1), name="dropout_residual_fp32"),
        # inside a wide feed-forward block, with its bias and activation: training
        dict(_dropout("dropout_train", 4, 4096, 8192, "bf16", "none", True, "gelu", 0.1), name="dropout_feed_forward"),
        # rows of an odd width, half-precision blocks onto a stream in fp32
        dict(_dropout("dropout_train", 7, 773, 1001, "bf16", "fp32", True, "relu", 0.5), name="dropout_odd_mixed"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm, odd as often as not."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["prefill", "train", "train", "step", "dropout", "dropout_train"])
    while True:
        if kind in ("dropout", "dropout_train"):
            case = _dropout(kind, _spread(rng, 1, 64), _spread(rng, 1, 8192), _spread(rng, 32, 8192),
                            rng.choice(["fp32", "bf16"]), rng.choice(["none", "fp32", "bf16"]), rng.choice([True, False]),
                            rng.choice(["none", "relu", "gelu", "silu"]), rng.choice([0.0, 0.05, 0.1, 0.2, 0.5, 0.9]))
        else:
            Hk = _spread(rng, 1, 16)
            H = Hk * rng.choice([1, 1, 2, 4])
            E = rng.choice([32, 64, 96, 128, _spread(rng, 8, 128)])
            M = rng.choice([32, 64, 128, 256, _spread(rng, 8, 256)])
            dtype, decay = rng.choice(["fp32", "bf16"]), rng.choice(["head", "position"])
            if kind == "step":
                case = _step(_spread(rng, 1, 256), H, Hk, E, M, dtype, decay)
            else:
                case = _rule(kind, _spread(rng, 1, 16), H, Hk, _spread(rng, 1, 16384), E, M, dtype, decay,
                             rng.choice([True, False]), kind == "train" and rng.choice([True, False]))
        w = work(case)
        if w["bytes"] <= 1.1e9 and w["flops"] <= 1.2e11:
            return case


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _decays(gen, case, row):
    """Log decays: one for each head, log(1 - 2^(-1 - x)) with x from nothing to eight, or of every position as such models
    make them, -exp(a) softplus(y), from a hundredth to a few."""
    H = case["H"]
    if case["decay"] == "head":
        return torch.log1p(-torch.exp2(-1 - 8 * torch.rand(H, generator=gen, device="cuda")))
    rates = torch.exp(-4 + 4 * torch.rand(H, generator=gen, device="cuda"))
    return -rates.view(1, -1, *[1] * len(row)) * torch.nn.functional.softplus(_randn(gen, case["N"], H, *row))


def _inputs_rule(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    N, H, Hk, E, M = (case[x] for x in ("N", "H", "Hk", "E", "M"))
    row = () if case["kind"] == "step" else (case["L"],)
    # projections lie as (N, L, heads, width) and are handed over as views
    turn = (lambda t: t) if case["kind"] == "step" else (lambda t: t.permute(0, 2, 1, 3))
    q, k = (turn(_randn(gen, N, *row, Hk, E).to(dtype)) for _ in range(2))
    v = turn(_randn(gen, N, *row, H, M).to(dtype))
    state = dict(q=q, k=k, v=v, g=_decays(gen, case, row), s0=_randn(gen, N, H, E, M), scale=E ** -0.5, lengths=None)
    if case.get("ragged"):
        lengths = torch.randint(0, case["L"] + 1, (N,), generator=gen, device="cuda")
        lengths[0] = case["L"]
        state["lengths"] = lengths
    if case["kind"] == "train":
        state["go"] = _randn(gen, N, H, case["L"], M).to(dtype)
        if not case["carry"]:
            state["s0"] = None
    return state


def _inputs_dropout(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    N, L, D = case["N"], case["L"], case["D"]
    stream = None if case["stream"] == "none" else _DTYPES[case["stream"]]
    s = dict(block=_randn(gen, N, L, D).to(dtype), residual=None, bias=None, seed=(seed * 0x9E3779B97F4A7C15 + 1) % 2 ** 63,
             offset=seed % 1000)
    if stream is not None:
        s["residual"] = (2 * _randn(gen, N, L, D)).to(stream)
    if case["bias"]:
        s["bias"] = 0.1 * _randn(gen, D)
    if case["kind"] == "dropout_train":
        s["gx"] = _randn(gen, N, L, D).to(stream or dtype)
    return s


_RULE_LEAVES = ("q", "k", "v", "g", "s0")
_DROPOUT_LEAVES = ("block", "residual", "bias")


def _leaves(case):
    return _DROPOUT_LEAVES if case["kind"] in ("dropout", "dropout_train") else _RULE_LEAVES


def prepare(case, seed):
    state = (_inputs_dropout if case["kind"] in ("dropout", "dropout_train") else _inputs_rule)(case, seed)
    if case["kind"] in ("train", "dropout_train"):
        for name in _leaves(case):
            if state[name] is not None:
                state[name].requires_grad_(True)
    state["case"] = case
    return state


# ---- the plain forms ----

def _plain_rule(q, k, v, g, s0, scale, lengths):
    """The attention in chunks of 64 positions, in fp32: everything inside the chunks at once, then the states one
    chunk after the other."""
    N, H, L, M = v.shape
    group, dtype = H // q.shape[1], v.dtype
    q, k = (t.float().repeat_interleave(group, 1) for t in (q, k))
    q, v = q * scale, v.float()
    g = (g[:, None].expand(N, H, L) if g.dim() == 1 else g).float()
    if lengths is not None:
        valid = (torch.arange(L, device=q.device) < lengths[:, None])[:, None]
        q, k, v = (torch.where(valid[..., None], t, 0.0) for t in (q, k, v))
        g = torch.where(valid, g, 0.0)
    pad = -L % _CHUNK
    C = (L + pad) // _CHUNK
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).reshape(N, H, C, _CHUNK, -1) for t in (q, k, v))
    G = torch.nn.functional.pad(g, (0, pad)).reshape(N, H, C, _CHUNK).double().cumsum(-1)  # (differences of long sums)
    lower = torch.tril(torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device))
    D = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~lower, 0.0).float())
    rise, fall, last = G.exp().float(), (G[..., -1:] - G).exp().float(), G[..., -1].exp().float()
    A = ((q @ k.transpose(-1, -2)) * D).masked_fill(~lower, 0.0)
    written = (k * fall[..., None]).transpose(-1, -2) @ v
    S = torch.zeros_like(written[:, :, 0]) if s0 is None else s0.float()
    states = []
    for c in range(C):
        states.append(S)
        S = last[:, :, c, None, None] * S + written[:, :, c]
    out = (rise[..., None] * q) @ torch.stack(states, 2) + A @ v
    return out.reshape(N, H, L + pad, M)[:, :, :L].to(dtype), S


def _plain_step(q, k, v, g, state, scale):
    group, dtype = v.shape[1] // q.shape[1], v.dtype
    q, k = (t.float().repeat_interleave(group, 1) for t in (q, k))
    S = state * torch.exp(g.float())[..., None, None] + k[..., None] * v.float()[..., None, :]
    state.copy_(S)
    return (S * (scale * q)[..., None]).sum(2).to(dtype)


def _plain_words(count, seed, offset, device):
    """The generator's first ``count`` words as whole numbers of 64 bits."""
    low = 0xFFFFFFFF
    at = torch.arange((count + 3) // 4, dtype=torch.int64, device=device)
    c = [at & low, at >> 32, torch.full_like(at, offset & low), torch.full_like(at, offset >> 32 & low)]
    key = [seed & low, seed >> 32 & low]
    for _ in range(10):
        # (products of 64 bits, wrapped: their halves are right all the same)
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32 & low) ^ c[1] ^ key[0], b & low, (a >> 32 & low) ^ c[3] ^ key[1], a & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    return torch.stack(c, -1).reshape(-1)[:count]


def _plain_dropout(s, case):
    block, p = s["block"], case["p"]
    a = block.float()
    if s["bias"] is not None:
        a = a + s["bias"]
    if case["activation"] == "relu":
        a = torch.where(a > 0, a, 0.0)
    elif case["activation"] == "gelu":
        a = 0.5 * a * (1 + torch.erf(a * math.sqrt(0.5)))
    elif case["activation"] == "silu":
        a = a / (1 + torch.exp(-a))
    keep = _plain_words(block.numel(), s["seed"], s["offset"], block.device).view(block.shape) >= round(p * 2 ** 32)
    x = torch.where(keep, a * (1 / (1 - p)), 0.0)
    if s["residual"] is not None:
        x = s["residual"].float() + x
    return x.to(block.dtype if s["residual"] is None else s["residual"].dtype)


# ---- one pass ----

@functools.lru_cache
def _package():
    root = os.path.abspath("fast-transformers_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from fast_transformers_amd import decayed_attention, dropout
    return decayed_attention, dropout


def _gradients(outs, grads, s, leaves):
    names = [n for n in leaves if s[n] is not None]
    return {"grad_" + n: t for n, t in zip(names, torch.autograd.grad(outs, [s[n] for n in names], grads))}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("dropout", "dropout_train"):
        if own:
            x = _package()[1].residual_dropout(
                s["block"], s["residual"], p=case["p"], seed=s["seed"], offset=s["offset"], bias=s["bias"],
                activation=None if case["activation"] == "none" else case["activation"])
        else:
            x = _plain_dropout(s, case)
        return {"x": x} if kind == "dropout" else {"x": x.detach(), **_gradients([x], [s["gx"]], s, _DROPOUT_LEAVES)}
    args = (s["q"], s["k"], s["v"], s["g"], s["s0"])
    if kind == "step":
        if own:
            out = _package()[0].decayed_attention_step(*args, scale=s["scale"])
        else:
            out = _plain_step(*args, s["scale"])
        return {"out": out, "state": s["s0"]}
    if own:
        out, state = _package()[0].decayed_attention(*args, scale=s["scale"], lengths=s["lengths"], return_state=True)
    else:
        out, state = _plain_rule(*args, s["scale"], s["lengths"])
    if kind == "prefill":
        return {"out": out, "state": state}
    return {"out": out.detach(), "state": state.detach(), **_gradients([out], [s["go"]], s, _RULE_LEAVES)}


def work(case):
    size = {"fp32": 4, "bf16": 2}
    b = size[case["dtype"]]
    if case["kind"] in ("dropout", "dropout_train"):
        values = case["N"] * case["L"] * case["D"]
        stream = b if case["stream"] == "none" else size[case["stream"]]
        residual = 0 if case["stream"] == "none" else stream
        # block and residual in, x out; ten rounds of two products for every four values, and the activation
        one, bias = values * (b + residual + stream), 4 * case["D"] * case["bias"]
        if case["kind"] == "dropout":
            return {"bytes": float(one + bias), "flops": 20.0 * values}
        # ... block and the gradient of x in, those of block, residual and bias out
        return {"bytes": float(2 * one + values * b + 2 * bias), "flops": 60.0 * values}
    N, H, Hk, E, M = (case[x] for x in ("N", "H", "Hk", "E", "M"))
    L = case.get("L", 1)
    decays = 4 * (H if case["decay"] == "head" else N * H * L)
    rows = N * L * (2 * Hk * E * b + 2 * H * M * b) + decays
    state = 4 * N * H * E * M
    flops = 5.0 * N * H * L * E * M  # the decay, the rank-one write, S^T q
    if case["kind"] == "train":
        # the state out; dO in and the gradients of q, k, v and g out, with q, k and v read again
        more = N * L * (4 * Hk * E * b + 3 * H * M * b) + decays
        return {"bytes": float(rows + more + (3 if case["carry"] else 1) * state), "flops": 3 * flops}
    return {"bytes": float(rows + 2 * state), "flops": flops}


# ---- the definition, in 64 bits ----

def _exact_rule(case, s):
    """One position after the other, forward, and backward with the states made again from every 64th."""
    kind, L = case["kind"], case["L"]
    N, H, Hk, E, M = (case[x] for x in ("N", "H", "Hk", "E", "M"))
    group, scale = H // Hk, s["scale"]
    by_position = lambda t: t.detach().double().permute(2, 0, 1, 3).contiguous()  # noqa: E731
    q, k = (by_position(s[n].detach().repeat_interleave(group, 1)) for n in ("q", "k"))
    v = by_position(s["v"])
    g = s["g"].detach().double()
    a = (g.exp()[None, None].expand(L, N, H) if g.dim() == 1 else g.exp().permute(2, 0, 1)).contiguous()
    live = torch.ones(L, N, 1, dtype=torch.float64, device=v.device)
    if s["lengths"] is not None:
        live = (torch.arange(L, device=v.device)[:, None] < s["lengths"]).double()[..., None]
        a = torch.where(live > 0, a, 1.0)
    q, k = q * live[..., None] * scale, k * live[..., None]
    S = torch.zeros(N, H, E, M, dtype=torch.float64, device=v.device) if s["s0"] is None else s["s0"].detach().double()
    o, kept = torch.empty_like(v), {}
    for t in range(L):
        if t % 64 == 0:
            kept[t] = S
        S = torch.addcmul(a[t][..., None, None] * S, k[t][..., :, None], v[t][..., None, :])
        o[t] = (q[t][..., None, :] @ S)[..., 0, :]
    result = {"out": o.permute(1, 2, 0, 3), "state": S}
    if kind == "prefill":
        return result
    go = by_position(s["go"])
    dq, dk, dv, dg = (torch.empty_like(t) for t in (q, k, v, a))
    dS = torch.zeros_like(S)
    for start in sorted(kept, reverse=True):
        before = [kept[start]]
        for t in range(start, min(L, start + 64)):
            before.append(torch.addcmul(a[t][..., None, None] * before[-1], k[t][..., :, None], v[t][..., None, :]))
        for t in range(min(L, start + 64) - 1, start - 1, -1):
            dq[t] = (before[t - start + 1] @ go[t][..., None])[..., 0]
            dS = torch.addcmul(dS, q[t][..., :, None], go[t][..., None, :])
            dk[t] = (dS @ v[t][..., None])[..., 0]
            dv[t] = (k[t][..., None, :] @ dS)[..., 0, :]
            dS = a[t][..., None, None] * dS
            dg[t] = (dS * before[t - start]).sum((-1, -2))
    heads = lambda t: (t * live[..., None]).permute(1, 2, 0, 3).reshape(N, Hk, group, L, E).sum(2)  # noqa: E731
    dg = (dg * live).permute(1, 2, 0)
    result.update(grad_q=heads(dq * scale), grad_k=heads(dk), grad_v=(dv * live[..., None]).permute(1, 2, 0, 3),
                  grad_g=dg.sum((0, 2)) if g.dim() == 1 else dg)
    if s["s0"] is not None:
        result["grad_s0"] = dS
    return result


def _exact_step(case, s):
    group = case["H"] // case["Hk"]
    q, k = (s[n].double().repeat_interleave(group, 1)[..., None, :] for n in ("q", "k"))
    state = s["s0"].double() * s["g"].double().exp()[..., None, None] + k.transpose(-1, -2) @ s["v"].double()[..., None, :]
    return {"out": s["scale"] * (q @ state)[..., 0, :], "state": state}


def _exact_keep(case, s):
    """Which values are kept, from the generator in whole numbers without a sign, four words at a time."""
    count = s["block"].numel()
    u32, u64 = numpy.uint32, numpy.uint64
    at = numpy.arange((count + 3) // 4, dtype=u64)
    x0, x1 = at.astype(u32), (at >> u64(32)).astype(u32)
    x2, x3 = (numpy.full(at.shape, s["offset"] >> shift & 0xFFFFFFFF, dtype=u32) for shift in (0, 32))
    for turn in range(10):
        k0, k1 = ((s["seed"] >> shift) + turn * step & 0xFFFFFFFF for shift, step in ((0, 0x9E3779B9), (32, 0xBB67AE85)))
        left, right = x0.astype(u64) * u64(0xD2511F53), x2.astype(u64) * u64(0xCD9E8D57)
        x0, x2 = (right >> u64(32)).astype(u32) ^ x1 ^ u32(k0), (left >> u64(32)).astype(u32) ^ x3 ^ u32(k1)
        x1, x3 = right.astype(u32), left.astype(u32)
    keep = numpy.stack([x.astype(u64) >= u64(round(case["p"] * 2 ** 32)) for x in (x0, x1, x2, x3)], -1).reshape(-1)[:count]
    return torch.from_numpy(keep).to(s["block"].device).view(s["block"].shape)


def _exact_dropout(case, s):
    # (by parts of the rows where there are many: 64 bits of several values each)
    keep, D = _exact_keep(case, s).view(-1, case["D"]), case["D"]
    flat = lambda t: None if t is None else t.detach().reshape(-1, D)  # noqa: E731
    block, residual, gx = flat(s["block"]), flat(s["residual"]), flat(s.get("gx"))
    parts, part = {}, 1 << 12
    for lo in range(0, block.shape[0], part):
        z = block[lo:lo + part].double() + (0 if s["bias"] is None else s["bias"].detach().double())
        if case["activation"] == "none":
            a, slope = z, torch.ones_like(z)
        elif case["activation"] == "relu":
            a, slope = z.clamp_min(0), (z > 0).double()
        elif case["activation"] == "gelu":
            phi = torch.special.ndtr(z)
            a, slope = z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        else:
            sigmoid = torch.sigmoid(z)
            a, slope = z * sigmoid, sigmoid * (1 + z * (1 - sigmoid))
        factor = keep[lo:lo + part].double() / (1 - case["p"])
        x = a * factor
        got = {"x": x if residual is None else x + residual[lo:lo + part].double()}
        if gx is not None:
            got["grad_block"] = factor * slope * gx[lo:lo + part].double()
        for name, t in got.items():
            parts.setdefault(name, []).append(t)
    shape = s["block"].shape
    out = {name: torch.cat(t).view(shape) for name, t in parts.items()}
    if gx is not None:
        if residual is not None:
            out["grad_residual"] = s["gx"].double()
        if s["bias"] is not None:
            out["grad_bias"] = out["grad_block"].sum((0, 1))
    return out


def exact(case, seed):
    if case["kind"] in ("dropout", "dropout_train"):
        return _exact_dropout(case, _inputs_dropout(case, seed))
    s = _inputs_rule(case, seed)
    return _exact_step(case, s) if case["kind"] == "step" else _exact_rule(case, s)
