"""Operators that are differentiated once, or not at all."""
import functools

import torch


class _NotDifferentiated(torch.autograd.Function):
    """The first tensors as they are, as functions of all that they were made of, whose own gradient is an error."""

    @staticmethod
    def forward(ctx, error, count, *tensors):
        ctx.error = error
        return tuple(t.clone() for t in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(ctx.error)


def not_differentiated(error, result, made_of):
    """``result`` where nothing that it was made of requires a gradient, else one whose gradient is an error."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in made_of):
        return _NotDifferentiated.apply(error, 1, result, *made_of)[0]
    return result


def check_factor(factor, what):
    """A factor that the kernels take as a number: a tensor's gradient would be lost."""
    if isinstance(factor, torch.Tensor) and factor.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(what + ": scale is a number, not a tensor that requires a gradient")


def differentiated_once(what):
    """Decorator of a Function's backward: where the gradients are to be differentiated again (``create_graph``), their
    own gradient is an error, also with respect to saved tensors (which torch's ``once_differentiable`` passes over)."""
    def wrap(backward):
        @functools.wraps(backward)
        def run(ctx, *grads):
            with torch.no_grad():
                out = list(backward(ctx, *grads))
            if torch.is_grad_enabled():
                there = [i for i, t in enumerate(out) if t is not None]
                made_of = [t for t in (*ctx.saved_tensors, *grads) if t is not None]
                for i, t in zip(there, _NotDifferentiated.apply(what + ": the gradients cannot be differentiated again", len(there),
                                                     *(out[i] for i in there), *made_of)):
                    out[i] = t
            return tuple(out)
        return run
    return wrap


__all__ = ["check_factor", "differentiated_once", "not_differentiated"]
