"""Linear attention with a decay for each head: the causal linear attention whose state fades.

Per chain of a value head, on a state ``S`` of ``E x M`` in float32 (``q``, ``k`` of ``E`` values, ``v`` of ``M``):

    S_l = exp(g_l) S_{l-1} + k_l v_l^T,  out_l = scale S_l^T q_l

With ``g = 0`` and ``scale = 1`` this is the sum that ``causal_dot_product`` computes; the gated delta rule
(``delta_rule``) corrects what it writes as well.

* ``decayed_attention``: whole sequences, or a piece of them with the state handed in and out, differentiable.
* ``decayed_attention_step``: one token of every sequence, the state updated in place.

On the GPU the HIP kernels run (``csrc/ftc_decay*.hip``); without the library a GPU tensor raises.  CPU tensors
take an implementation of their own in torch operations, which shares nothing with the kernels.
"""
import torch

from .. import _native
from .._once import check_factor, differentiated_once, not_differentiated

_CPU_CHUNK = 32


def _check(queries, keys, values, log_decay, state, what):
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
    for name, t in (("queries", queries), ("log_decay", log_decay)):
        if t.dtype not in (torch.float32, torch.bfloat16):
            raise RuntimeError("%s: %s must be float32 or bfloat16, got %s" % (what, name, t.dtype))
    if log_decay.shape not in (values.shape[:-1], values.shape[1:2]):
        raise RuntimeError("%s: log_decay must have shape %s or %s, got %s"
                           % (what, tuple(values.shape[:-1]), tuple(values.shape[1:2]), tuple(log_decay.shape)))
    if not (1 <= queries.shape[-1] <= 128 and 1 <= values.shape[-1] <= 512):
        raise RuntimeError("%s: takes key rows of 1 to 128 values and value rows of 1 to 512, got %d and %d"
                           % (what, queries.shape[-1], values.shape[-1]))
    if state is not None and (state.dtype != torch.float32 or tuple(state.shape) != (
            values.shape[0], values.shape[1], queries.shape[-1], values.shape[-1])):
        raise RuntimeError("%s: the state must be a float32 tensor of shape (N, H, E, M)" % what)
    for t in (keys, values, log_decay, state):
        if t is not None and t.device != queries.device:
            raise RuntimeError("%s: all tensors must be on one device" % what)


class DecayedAttention(torch.autograd.Function):
    """``(out, final_state)`` on the GPU and their gradients, tensors in the ``(N, H, L, X)`` layout.  Plain calls run as
    the same function of the C++ engine (``host/ftc_host.cpp``), which costs the host less; calls that are watched or
    transformed run this one."""

    @staticmethod
    def forward(ctx, queries, keys, values, log_decay, initial_state, lengths, scale):
        out, state, kept = _native.host().decayed_attention(queries, keys, values, log_decay, initial_state, lengths, scale,
                                                            True, True)
        ctx.save_for_backward(queries, keys, values, log_decay, initial_state, kept, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @differentiated_once("decayed_attention")
    def backward(ctx, grad_out, grad_state):
        queries, keys, values, log_decay, initial_state, kept, lengths = ctx.saved_tensors
        if values.shape[2] == 0:
            grads = [torch.zeros_like(t) if need else None for t, need in zip(
                (queries, keys, values, log_decay), ctx.needs_input_grad)]
            return (*grads, grad_state if ctx.needs_input_grad[4] else None, None, None)
        if grad_out is None:
            grad_out = torch.zeros_like(values)
        grads = _native.host().decayed_attention_backward(
            queries, keys, values, log_decay, initial_state, lengths, ctx.scale, kept, grad_out, grad_state,
            list(ctx.needs_input_grad[:5]))
        return (*grads, None, None)


def _cpu_attention(queries, keys, values, log_decay, state, lengths, scale):
    """CPU tensors: chunks of positions in float32; autograd differentiates it."""
    N, H, L, M = values.shape
    group = H // max(1, queries.shape[1])
    g = log_decay.float().clamp_min(-1000.0)
    if g.dim() == 1:
        g = g[:, None].expand(N, H, L)
    if lengths is not None:  # (before anything is made of them: gradients of what is masked afterwards may be 0 x NaN)
        valid = (torch.arange(L, device=values.device) < lengths[:, None])[:, None]
        queries, keys, values = (torch.where(valid[..., None], t, 0.0) for t in (queries, keys, values))
        g = torch.where(valid, g, 0.0)
    q, k = (t.float().repeat_interleave(group, 1) for t in (queries, keys))
    v = values.float()
    S = v.new_zeros((N, H, q.shape[3], M)) if state is None else state
    outs = []
    for lo in range(0, L, _CPU_CHUNK):
        qc, kc, vc, gc = (t[:, :, lo:lo + _CPU_CHUNK] for t in (q, k, v, g))
        G = gc.double().cumsum(-1)
        keep = torch.tril(torch.ones(G.shape[-1], G.shape[-1], dtype=torch.bool))
        D = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~keep, 0.0)).float()
        rise, fall = G.exp().float()[..., None], (G[..., -1:] - G).exp().float()[..., None]
        A = (torch.matmul(qc, kc.transpose(-1, -2)) * D).masked_fill(~keep, 0.0)
        outs.append(scale * (rise * torch.matmul(qc, S) + torch.matmul(A, vc)))
        S = rise[:, :, -1:] * S + torch.matmul((fall * kc).transpose(-1, -2), vc)
    out = torch.cat(outs, 2) if outs else v.new_zeros((N, H, 0, M))
    if lengths is not None:  # (a state or a row without numbers does not reach them, nor their gradients what is before)
        out = torch.where(valid[..., None], out, 0.0)
    return out.to(values.dtype), S if outs or state is None else S.clone()


def decayed_attention(queries, keys, values, log_decay, initial_state=None, *, scale=None, lengths=None, return_state=False):
    """The attention over whole sequences.

    ``queries``, ``keys``: ``(N, Hk, L, E)``; ``values``: ``(N, H, L, M)`` of the same type (float32 or bfloat16; any
    strides, permuted views of ``(N, L, H, X)`` projections are read where they lie); value head ``h`` reads key head
    ``h // (H // Hk)``.  ``log_decay``, float32 or bfloat16: ``(N, H, L)``, one of every position, or ``(H,)``, one for each
    head; a decay of ``-inf`` forgets the state.  ``initial_state``: ``(N, H, E, M)`` float32, or None for zeros.  ``scale``:
    factor of the queries, ``E ** -0.5`` by default.  ``lengths``: None, or an int64 tensor of N lengths: positions past them
    leave the state as it is, are not looked at, and have outputs and gradients of zero.

    Returns the outputs, ``(N, H, L, M)`` in the values' type, and with ``return_state`` also the state after the
    last position, float32.  E is at most 128, M at most 512; N H ceil(M / 128) is below 2^21 on the GPU, and in
    a call that will be differentiated below 2^20 and, times ceil(L / 1024), below 2^22.
    Differentiable once, in reverse, with respect to everything
    but ``lengths`` and ``scale``; a call that will be differentiated keeps the states every 1024 positions or fewer.  Log decays are
    meant to be at most zero; the gradient of one of ``-inf`` is zero.  Chunks of positions are worked on as a whole: NaN or infinity in a
    row within its length also reaches the outputs of up to 63 positions before it."""
    if queries.dim() != 4:
        raise RuntimeError("decayed_attention: expected queries (N, Hk, L, E), got %s" % (tuple(queries.shape),))
    if queries.device.type != "cuda":  # (the native code checks for itself)
        _check(queries, keys, values, log_decay, initial_state, "decayed_attention")
    if scale is None:
        scale = max(1, queries.shape[3]) ** -0.5
    elif queries.device.type == "cuda":
        check_factor(scale, "decayed_attention")
    if lengths is not None:
        if lengths.shape != values.shape[:1]:
            raise RuntimeError("decayed_attention: expected %d lengths, got shape %s" % (values.shape[0], tuple(lengths.shape)))
        lengths = lengths.to(device=queries.device, dtype=torch.int64).contiguous()
    if queries.device.type != "cuda":
        out, state = _cpu_attention(queries, keys, values, log_decay, initial_state, lengths, scale)
    elif (torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (queries, keys, values, log_decay, initial_state))
            or torch.jit.is_tracing()):  # (a tracer sees the function)
        args = (queries, keys, values, log_decay, initial_state, lengths, scale)
        out, state = (None if torch.compiler.is_compiling() else _native.host().decayed_attention_plain(*args)) or \
            DecayedAttention.apply(*args)
    else:
        out, state, _ = _native.host().decayed_attention(queries, keys, values, log_decay, initial_state, lengths, scale,
                                                         return_state, False)
    return (out, state) if return_state else out


def decayed_attention_step(queries, keys, values, log_decay, state, *, scale=None):
    """One token of every sequence: ``queries``, ``keys`` ``(N, Hk, E)``, ``values`` ``(N, H, M)``, ``log_decay`` ``(N, H)`` or
    ``(H,)``; ``state`` ``(N, H, E, M)`` float32, updated in place (views of a larger buffer are fine, rows along M
    contiguous).  Returns the outputs ``(N, H, M)`` in the values' type, whose gradient is an error; one launch.  On the GPU
    N H ceil(M / 64) is below 2^22."""
    if queries.dim() != 3:
        raise RuntimeError("decayed_attention_step: expected queries (N, Hk, E), got %s" % (tuple(queries.shape),))
    on_gpu = queries.device.type == "cuda"
    if not on_gpu:  # (the native code checks for itself)
        _check(queries, keys, values, log_decay, state, "decayed_attention_step")
    if state.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("decayed_attention_step: the state is updated in place and cannot be differentiated")
    if scale is None:
        scale = max(1, queries.shape[2]) ** -0.5
    elif on_gpu:
        check_factor(scale, "decayed_attention_step")
    if not on_gpu:
        reach = state.shape[3]
        for stride, size in sorted(zip(state.stride()[:3], state.shape[:3])):
            if size > 1 and stride < reach:
                raise RuntimeError("decayed_attention_step: state is written and must not overlap itself")
            reach += stride * (size - 1)
        with torch.no_grad():
            decays = log_decay if log_decay.dim() == 1 else log_decay.unsqueeze(2)
            out, after = _cpu_attention(*(t.unsqueeze(2) for t in (queries, keys, values)), decays, state, None, scale)
            state.copy_(after)
        return not_differentiated("decayed_attention_step: the result cannot be differentiated", out.squeeze(2),
                                  (queries, keys, values, log_decay))
    return _native.host().decayed_step(queries, keys, values, log_decay, state, scale)
