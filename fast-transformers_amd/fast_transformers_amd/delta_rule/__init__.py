"""The gated delta rule: causal linear attention whose state fades and whose writes correct it.

Per chain of a value head, on a state ``S`` of ``E x M`` in float32 (``q``, ``k`` of ``E`` values, ``v`` of ``M``):

    S' = exp(g_l) S_{l-1},  z_l = v_l - S'^T k_l,  S_l = S' + k_l (beta_l z_l)^T,  out_l = scale S_l^T q_l

With ``g = 0`` and without the correction this is the sum that ``causal_dot_product`` computes.

* ``gated_delta_rule``: whole sequences, or a piece of them with the state handed in and out, differentiable.
* ``gated_delta_step``: one token of every sequence, the state updated in place.

On the GPU the HIP kernels run (``csrc/ftc_delta*.hip``); without the library a GPU tensor raises.  CPU tensors
take an implementation of their own in torch operations, which shares nothing with the kernels.
"""
import torch

from .. import _native
from .._once import check_factor, differentiated_once, not_differentiated

_EPS = 1e-6
_CPU_CHUNK = 32


def _check(queries, keys, values, log_decay, beta, state, what):
    """Shapes and types of a call on CPU tensors."""
    if queries.dim() != values.dim() or keys.shape != queries.shape or \
            queries.shape[0] != values.shape[0] or queries.shape[2:-1] != values.shape[2:-1]:
        raise RuntimeError("%s: expected queries and keys of one shape and values that fit them, got %s, %s and %s"
                           % (what, tuple(queries.shape), tuple(keys.shape), tuple(values.shape)))
    if values.shape[1] and (queries.shape[1] == 0 or values.shape[1] % queries.shape[1]):
        raise RuntimeError("%s: the number of value heads (%d) must be a multiple of the number of key heads (%d)"
                           % (what, values.shape[1], queries.shape[1]))
    if not queries.dtype == keys.dtype == values.dtype:
        raise RuntimeError("%s: queries, keys and values must have one type, got %s, %s and %s"
                           % (what, queries.dtype, keys.dtype, values.dtype))
    for name, t in (("queries", queries), ("log_decay", log_decay), ("beta", beta)):
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise RuntimeError("%s: %s must be float32 or bfloat16, got %s" % (what, name, t.dtype))
    for name, t in (("log_decay", log_decay), ("beta", beta)):
        if t.shape != values.shape[:-1]:
            raise RuntimeError("%s: %s must have shape %s, got %s"
                               % (what, name, tuple(values.shape[:-1]), tuple(t.shape)))
    if not (1 <= queries.shape[-1] <= 128 and 1 <= values.shape[-1] <= 512):
        raise RuntimeError("%s: takes key rows of 1 to 128 values and value rows of 1 to 512, got %d and %d"
                           % (what, queries.shape[-1], values.shape[-1]))
    if state is not None and (state.dtype != torch.float32 or tuple(state.shape) != (
            values.shape[0], values.shape[1], queries.shape[-1], values.shape[-1])):
        raise RuntimeError("%s: the state must be a float32 tensor of shape (N, H, E, M)" % what)
    for t in (keys, values, log_decay, beta, state):
        if t is not None and t.device != queries.device:
            raise RuntimeError("%s: all tensors must be on one device" % what)


class GatedDeltaRule(torch.autograd.Function):
    """``(out, final_state)`` on the GPU and their gradients, tensors in the ``(N, H, L, X)`` layout.  Plain calls run as
    the same function of the C++ engine (``host/ftc_host.cpp``), which costs the host less; calls that are watched or
    transformed run this one."""

    @staticmethod
    def forward(ctx, queries, keys, values, log_decay, beta, initial_state, lengths, scale, normalize):
        out, state, kept = _native.host().delta_rule(
            queries, keys, values, log_decay, beta, initial_state, lengths, scale, normalize, True, True)
        ctx.save_for_backward(queries, keys, values, log_decay, beta, kept, lengths)
        ctx.scale, ctx.normalize = scale, normalize
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @differentiated_once("gated_delta_rule")
    def backward(ctx, grad_out, grad_state):
        queries, keys, values, log_decay, beta, kept, lengths = ctx.saved_tensors
        if values.shape[2] == 0:
            grads = [torch.zeros_like(t) if need else None for t, need in zip(
                (queries, keys, values, log_decay, beta), ctx.needs_input_grad)]
            return (*grads, grad_state if ctx.needs_input_grad[5] else None, None, None, None)
        if grad_out is None:
            grad_out = torch.zeros_like(values)
        grads = _native.host().delta_rule_backward(
            queries, keys, values, log_decay, beta, lengths, ctx.scale, ctx.normalize, kept, grad_out, grad_state,
            list(ctx.needs_input_grad[:6]))
        return (*grads, None, None, None)


def _unit(x, normalize):
    if not normalize:
        return x
    x = x.double()  # (of a row of one value the gradient leaves eps / (x^2 + eps) of what it is a difference of)
    return (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + _EPS)).float()


def _solve_lower(strict, rows):
    """(I + strict)^-1 rows by substitution, row after row."""
    done = []
    for i in range(strict.shape[-1]):
        row = rows[..., i, :]
        if done:
            row = row - (strict[..., i, :i, None] * torch.stack(done, -2)).sum(-2)
        done.append(row)
    return torch.stack(done, -2)


def _cpu_rule(queries, keys, values, log_decay, beta, state, lengths, scale, normalize):
    """CPU tensors: chunks of positions, each solved for its writes, in float32; autograd differentiates it."""
    N, H, L, M = values.shape
    group = H // max(1, queries.shape[1])
    if lengths is not None:  # (before anything is made of them: gradients of what is masked afterwards may be 0 x NaN)
        valid = (torch.arange(L, device=values.device) < lengths[:, None])[:, None]
        queries, keys, values = (torch.where(valid[..., None], t, 0.0) for t in (queries, keys, values))
        log_decay, beta = (torch.where(valid, t, 0.0) for t in (log_decay, beta))
    q, k = (_unit(t.float(), normalize).repeat_interleave(group, 1) for t in (queries, keys))
    v, g, b = values.float(), log_decay.float().clamp_min(-1000.0), beta.float()
    S = v.new_zeros((N, H, q.shape[3], M)) if state is None else state
    outs = []
    for lo in range(0, L, _CPU_CHUNK):
        qc, kc, vc, gc, bc = (t[:, :, lo:lo + _CPU_CHUNK] for t in (q, k, v, g, b))
        G = gc.double().cumsum(-1)
        C = G.shape[-1]
        keep = torch.tril(torch.ones(C, C, dtype=torch.bool))
        D = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~keep, 0.0)).float()
        rise, fall = G.exp().float()[..., None], (G[..., -1:] - G).exp().float()[..., None]
        M_ = (torch.matmul(kc, kc.transpose(-1, -2)) * D * bc[..., None, :]).masked_fill(~torch.tril(keep, -1), 0.0)
        z = _solve_lower(M_, vc - rise * torch.matmul(kc, S))
        u = bc[..., None] * z
        A = (torch.matmul(qc, kc.transpose(-1, -2)) * D).masked_fill(~keep, 0.0)
        outs.append(scale * (rise * torch.matmul(qc, S) + torch.matmul(A, u)))
        S = rise[:, :, -1:] * S + torch.matmul((fall * kc).transpose(-1, -2), u)
    out = torch.cat(outs, 2) if outs else v.new_zeros((N, H, 0, M))
    if lengths is not None:
        out = torch.where(valid[..., None], out, 0.0)
    return out.to(values.dtype), S if outs or state is None else S.clone()


def gated_delta_rule(queries, keys, values, log_decay, beta, initial_state=None, *, scale=None, normalize=False,
                     lengths=None, return_state=False):
    """The rule over whole sequences.

    ``queries``, ``keys``: ``(N, Hk, L, E)``; ``values``: ``(N, H, L, M)`` of the same type (float32 or bfloat16; any
    strides, permuted views of ``(N, L, H, X)`` projections are read where they lie); value head ``h`` reads key head
    ``h // (H // Hk)``.  ``log_decay``, ``beta``: ``(N, H, L)``, float32 or bfloat16; a decay of ``-inf`` forgets the
    state.  ``initial_state``: ``(N, H, E, M)`` float32, or None for zeros.  ``scale``: factor of the queries,
    ``E ** -0.5`` by default.  ``normalize``: queries and keys are divided by ``sqrt(|x|^2 + 1e-6)``.
    ``lengths``: None, or an int64 tensor of N lengths: positions past them leave the state as it is, are not looked
    at, and have outputs and gradients of zero.

    Returns the outputs, ``(N, H, L, M)`` in the values' type, and with ``return_state`` also the state after the
    last position, float32.  E is at most 128, M at most 512.  Differentiable once, in reverse, with respect to everything
    but ``lengths``, ``scale`` and ``normalize``; a call that will be differentiated keeps the states
    before every 64th position and what the chunks were solved with: 3 KB a position and value head at E = M = 128 in
    bfloat16, 2 KB at 64 in float32.  Log decays are meant to be at most zero.  A ``beta`` of zero writes nothing (in
    gradients, nor does one of up to ``2 ** -64`` in size)."""
    if queries.dim() != 4:
        raise RuntimeError("gated_delta_rule: expected queries (N, Hk, L, E), got %s" % (tuple(queries.shape),))
    if queries.device.type != "cuda":  # (the native code checks for itself)
        _check(queries, keys, values, log_decay, beta, initial_state, "gated_delta_rule")
    if scale is None:
        scale = max(1, queries.shape[3]) ** -0.5
    elif queries.device.type == "cuda":
        check_factor(scale, "gated_delta_rule")
    if lengths is not None:
        if lengths.shape != values.shape[:1]:
            raise RuntimeError("gated_delta_rule: expected %d lengths, got shape %s"
                               % (values.shape[0], tuple(lengths.shape)))
        lengths = lengths.to(device=queries.device, dtype=torch.int64).contiguous()
    if queries.device.type != "cuda":
        out, state = _cpu_rule(queries, keys, values, log_decay, beta, initial_state, lengths, scale, normalize)
    elif (torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (queries, keys, values, log_decay, beta, initial_state))
            or torch.jit.is_tracing()):  # (a tracer sees the function)
        args = (queries, keys, values, log_decay, beta, initial_state, lengths, scale, normalize)
        out, state = (None if torch.compiler.is_compiling() else _native.host().delta_rule_plain(*args)) or \
            GatedDeltaRule.apply(*args)
    else:
        out, state, _ = _native.host().delta_rule(queries, keys, values, log_decay, beta, initial_state, lengths, scale,
                                                  normalize, return_state, False)
    return (out, state) if return_state else out


def gated_delta_step(queries, keys, values, log_decay, beta, state, *, scale=None, normalize=False):
    """One token of every sequence: ``queries``, ``keys`` ``(N, Hk, E)``, ``values`` ``(N, H, M)``, ``log_decay``,
    ``beta`` ``(N, H)``; ``state`` ``(N, H, E, M)`` float32, updated in place (views of a larger buffer are fine, rows
    along M contiguous).  Returns the outputs ``(N, H, M)`` in the values' type, whose gradient is an error; one launch."""
    if queries.dim() != 3:
        raise RuntimeError("gated_delta_step: expected queries (N, Hk, E), got %s" % (tuple(queries.shape),))
    on_gpu = queries.device.type == "cuda"
    if not on_gpu:  # (the native code checks for itself)
        _check(queries, keys, values, log_decay, beta, state, "gated_delta_step")
    if state.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("gated_delta_step: the state is updated in place and cannot be differentiated")
    if scale is None:
        scale = max(1, queries.shape[2]) ** -0.5
    elif on_gpu:
        check_factor(scale, "gated_delta_step")
    if not on_gpu:
        reach = state.shape[3]
        for stride, size in sorted(zip(state.stride()[:3], state.shape[:3])):
            if size > 1 and stride < reach:
                raise RuntimeError("gated_delta_step: state is written and must not overlap itself")
            reach += stride * (size - 1)
        with torch.no_grad():
            out, after = _cpu_rule(*(t.unsqueeze(2) for t in (queries, keys, values, log_decay, beta)), state, None,
                                   scale, normalize)
            state.copy_(after)
        return not_differentiated("gated_delta_step: the result cannot be differentiated", out.squeeze(2),
                                  (queries, keys, values, log_decay, beta))
    return _native.host().delta_step(queries, keys, values, log_decay, beta, state, scale, normalize)
