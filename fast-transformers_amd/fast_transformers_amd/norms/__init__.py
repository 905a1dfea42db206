"""The norms around a block with its gate and residual scale, one pass over the rows.

    y = norm_after(block),   x = residual + scale act(gate) y,   h = norm_before(x)

``x`` is the residual stream behind the block and ``h`` what the next block reads.  Without a residual and a
``before`` this is the gated norm of an attention's heads.  On the GPU it is one HIP kernel forward and two backward
(``csrc/ftc_norm.hip``); without the library a GPU tensor raises.  CPU tensors take torch operations.
"""
import torch

from .. import _native
from .._once import check_factor, differentiated_once

_KINDS = {"rms": 1, "layer": 2}
_ACTIVATIONS = {None: 0, "sigmoid": 1, "silu": 2}
_TYPES = (torch.float32, torch.bfloat16)


def _norm(spec, width, name):
    """(kind, weight, bias) of ``("rms" or "layer"[, weight[, bias]])`` or None."""
    if spec is None:
        return 0, None, None
    spec = tuple(spec) if not isinstance(spec, str) else (spec,)
    if not 1 <= len(spec) <= 3 or spec[0] not in _KINDS:
        raise RuntimeError('residual_norm: %s must be None or ("rms" or "layer", weight, bias), got %r'
                           % (name, spec[:1]))
    kind, weight, bias = spec + (None,) * (3 - len(spec))
    for t in (weight, bias):
        if t is not None and (tuple(t.shape) != (width,) or t.dtype not in _TYPES):
            raise RuntimeError("residual_norm: the weight and bias of %s must be float32 or bfloat16 vectors of %d values"
                               % (name, width))
    return _KINDS[kind], weight, bias


def _gate_rows(gate, shape):
    """The gate as rows that serve whole runs of the block's rows: the dimensions that it has in full come first.
    One that does not lie that way is expanded (autograd sums its gradient)."""
    if gate.dim() > len(shape) or any(g not in (1, s) for g, s in zip(reversed(gate.shape), reversed(shape))) or \
            gate.dim() == 0 or gate.shape[-1] != shape[-1]:
        raise RuntimeError("residual_norm: a gate of shape %s does not fit a block of shape %s"
                           % (tuple(gate.shape), tuple(shape)))
    lead = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape[:-1])
    full = 0
    while full < len(lead) and lead[full] == shape[full]:
        full += 1
    if any(n != 1 for n in lead[full:]):
        gate = gate.expand(shape)
    return gate


class ResidualNorm(torch.autograd.Function):
    """``(x, h)`` on the GPU and their gradients; ``h`` is None without a norm before the next block.  Plain calls run as
    the same function of the C++ engine (``host/ftc_host.cpp``); calls that are watched or transformed, and those whose gate lies
    across the rows, run this one."""

    @staticmethod
    def forward(ctx, block, residual, gate, after_weight, after_bias, before_weight, before_bias, options):
        after, before, activation, scale, eps = options
        x, h, stats = _native.host().residual_norm(block, residual, gate, after, after_weight, after_bias, before,
                                                   before_weight, before_bias, activation, scale, eps, True)
        ctx.save_for_backward(block, residual, gate, after_weight, after_bias, before_weight, before_bias, stats)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return x, h

    @staticmethod
    @differentiated_once("residual_norm")
    def backward(ctx, grad_x, grad_h):
        block, residual, gate, aw, ab, bw, bb, stats = ctx.saved_tensors
        after, before, activation, scale, eps = ctx.options
        grads = _native.host().residual_norm_backward(
            block, residual, gate, after, aw, ab, before, bw, bb, activation, scale, eps, stats, grad_x, grad_h,
            list(ctx.needs_input_grad[:7]))
        return (*grads, None)


def _cpu_norm(x, kind, weight, bias, eps):
    if kind == 0:
        return x
    if kind == 2:
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        x = x * weight.float()
    return x if bias is None else x + bias.float()


def _cpu_residual_norm(block, residual, gate, after, before, activation, scale, eps):
    y = _cpu_norm(block.float(), *after, eps)
    if gate is not None:
        g = gate.float()
        y = y * (g if activation == 0 else torch.sigmoid(g) if activation == 1 else torch.nn.functional.silu(g))
    x = scale * y if residual is None else residual.float() + scale * y
    h = _cpu_norm(x, *before, eps).to(block.dtype) if before[0] else None
    return x.to(block.dtype if residual is None else residual.dtype), h


def residual_norm(block, residual=None, gate=None, *, after=None, before=None, scale=1.0, activation=None, eps=1e-6):
    """``(x, h)``: the stream behind a block, ``x = residual + scale act(gate) norm_after(block)``, and what the
    next block reads, ``h = norm_before(x)`` (None without ``before``).

    ``block``: rows of up to 16384 values (at least 3 where a norm is taken), float32 or bfloat16, in any number of dimensions; ``residual``: None, or
    of the block's shape in either type (``x`` has the residual's type, or the block's without one; ``h`` the
    block's); ``gate``: None, or of either type in a shape that broadcasts to the block's over all but the last
    dimension.  ``after``, ``before``: None, or ``("rms" or "layer", weight, bias)`` with weight and bias optional.
    ``activation`` of the gate: None, ``"sigmoid"`` or ``"silu"``.  ``h`` is the norm of ``x`` before ``x`` is rounded to its type.
    Differentiable once, in reverse, with respect to all tensors."""
    if type(scale) is not float and block.is_cuda:
        check_factor(scale, "residual_norm")
    if block.is_cuda and not torch.compiler.is_compiling():  # (calls as they mostly are, checked by the native code)
        pair = _native.host().residual_norm_plain(block, residual, gate, after, before, scale, activation, eps)
        if pair is not None:
            return pair
    if block.dim() < 1 or not 1 <= block.shape[-1] <= 16384:
        raise RuntimeError("residual_norm: takes rows of 1 to 16384 values, got shape %s" % (tuple(block.shape),))
    if activation not in _ACTIVATIONS:
        raise RuntimeError('residual_norm: activation must be None, "sigmoid" or "silu", got %r' % (activation,))
    for name, t in (("block", block), ("residual", residual), ("gate", gate)):
        if t is not None and t.dtype not in _TYPES:
            raise RuntimeError("residual_norm: %s must be float32 or bfloat16, got %s" % (name, t.dtype))
    if residual is not None and residual.shape != block.shape:
        raise RuntimeError("residual_norm: the residual has shape %s, the block %s"
                           % (tuple(residual.shape), tuple(block.shape)))
    after = _norm(after, block.shape[-1], "after")
    before = _norm(before, block.shape[-1], "before")
    if block.shape[-1] < 3 and (after[0] or before[0]):
        raise RuntimeError("residual_norm: rows of at least 3 values are normalised, got %d" % block.shape[-1])
    tensors = (block, residual, gate) + after[1:] + before[1:]
    if any(t is not None and t.device != block.device for t in tensors):
        raise RuntimeError("residual_norm: all tensors must be on one device")
    if gate is not None:
        gate = _gate_rows(gate, block.shape)
    activation = _ACTIVATIONS[activation]
    if block.device.type == "cpu":
        return _cpu_residual_norm(block, residual, gate, after, before, activation, scale, eps)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
            or torch.jit.is_tracing()):  # (a tracer sees the function)
        return ResidualNorm.apply(block, residual, gate, after[1], after[2], before[1], before[2],
                                  (after[0], before[0], activation, scale, eps))
    x, h, _ = _native.host().residual_norm(block, residual, gate, *after, *before, activation, scale, eps, False)
    return x, h
