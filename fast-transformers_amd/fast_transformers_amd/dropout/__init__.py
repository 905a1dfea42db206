"""The dropout behind a block with the block's bias, activation and residual, one pass over the rows.

    x = residual + keep act(block + bias) / (1 - p)

No mask is stored: whether value ``i`` is kept, counted over the block's values in the order of its shape, is a function of the
seed, the offset and ``i``, and the backward makes it again.  It is word ``i % 4`` of Philox4x32-10 (Salmon, Moraes, Dror and
Shaw, 2011) with the seed as its key and ``(i // 4, offset)`` as its counter, against ``p 2^32``.  On the GPU it is one HIP kernel
forward and one or two backward (``csrc/ftc_dropout.hip``); without the library a GPU tensor
raises.  CPU tensors take torch operations, with the same values kept.
"""
from operator import index

import torch

from .. import _native
from .._once import differentiated_once

_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}
_TYPES = (torch.float32, torch.bfloat16)
_ALL = 1 << 32
_LOW = 0xFFFFFFFF


class ResidualDropout(torch.autograd.Function):
    """``x`` on the GPU and its gradients.  Plain calls run as the same function of the C++ engine
    (``host/ftc_host.cpp``); calls that are watched or transformed run this one."""

    @staticmethod
    def forward(ctx, block, residual, bias, seeds, options):
        x = _native.host().residual_dropout(block, residual, bias, seeds, *options)
        ctx.save_for_backward(block if options[0] else None, bias, seeds)  # (without an activation only its type is needed)
        ctx.options, ctx.block_type = options, block.dtype
        ctx.set_materialize_grads(False)
        return x

    @staticmethod
    def backward(ctx, grad_x):
        if grad_x is None:
            return (None,) * 5
        grad_block, grad_bias = ResidualDropout._gradients(ctx, grad_x)
        return grad_block, grad_x if ctx.needs_input_grad[1] else None, grad_bias, None, None

    @staticmethod
    @differentiated_once("residual_dropout")
    def _gradients(ctx, grad_x):
        block, bias, seeds = ctx.saved_tensors
        needs_block, _, needs_bias = ctx.needs_input_grad[:3]
        if not (needs_block or needs_bias):
            return None, None
        return _native.host().residual_dropout_backward(block, ctx.block_type, bias, seeds, grad_x, *ctx.options, needs_block, needs_bias)


def _cpu_words(count, seed, offset):
    """The generator's first ``count`` words."""
    at = torch.arange((count + 3) // 4, dtype=torch.int64)
    c0, c1 = at & _LOW, at >> 32
    c2, c3 = (torch.full_like(at, offset >> shift & _LOW) for shift in (0, 32))
    k0, k1 = seed & _LOW, seed >> 32 & _LOW
    for _ in range(10):
        # (products of 64 bits, wrapped: their halves are right all the same)
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & _LOW) ^ c1 ^ k0, b & _LOW, (a >> 32 & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = k0 + 0x9E3779B9 & _LOW, k1 + 0xBB67AE85 & _LOW
    return torch.stack((c0, c1, c2, c3), -1).reshape(-1)[:count]


def _cpu_dropout(block, residual, bias, seeds, activation, dropped, seed, offset):
    if seeds is not None:
        seed, offset = (int(n) & (1 << 64) - 1 for n in seeds)
    keep = _cpu_words(block.numel(), seed, offset).view(block.shape) >= dropped
    z = block.float() if bias is None else block.float() + bias.float()
    z = torch.where(keep, z, 0.0)  # (before anything is made of them: gradients of what is dropped afterwards may be 0 x NaN)
    if activation == 2:  # (torch's gelu takes 1 + erf, which loses the tail)
        z = z * (0.5 * torch.special.erfc(z * -(0.5 ** 0.5)))
    else:
        z = {0: lambda t: t, 1: torch.relu, 3: torch.nn.functional.silu}[activation](z)
    x = torch.where(keep, z * (_ALL / max(1, _ALL - dropped)), 0.0)
    return (x if residual is None else residual.float() + x).to(block.dtype if residual is None else residual.dtype)


def _check(block, residual, bias):
    """Shapes and types of a call on CPU tensors."""
    if block.dim() < 1 or not 1 <= block.shape[-1] <= 1 << 18:
        raise RuntimeError("residual_dropout: takes rows of 1 to 262144 values, got shape %s" % (tuple(block.shape),))
    for name, t in (("block", block), ("residual", residual), ("bias", bias)):
        if t is not None and t.dtype not in _TYPES:
            raise RuntimeError("residual_dropout: %s must be float32 or bfloat16, got %s" % (name, t.dtype))
    if residual is not None and residual.shape != block.shape:
        raise RuntimeError("residual_dropout: the residual has shape %s, the block %s" % (tuple(residual.shape), tuple(block.shape)))
    if bias is not None and tuple(bias.shape) != (block.shape[-1],):
        raise RuntimeError("residual_dropout: the bias has shape %s, expected (%d,)" % (tuple(bias.shape), block.shape[-1]))


def residual_dropout(block, residual=None, *, p, seed, offset=0, bias=None, activation=None):
    """``x = residual + keep act(block + bias) / (1 - p)``, the stream behind a block whose values are dropped with
    probability ``p``.

    ``block``: rows of up to 262144 values, float32 or bfloat16, in any number of dimensions; ``residual``: None, or of the block's
    shape in either type (``x`` has the residual's type, or the block's without one); ``bias``: None, or a vector of the rows' width
    in either type.  ``activation``: None, ``"relu"``, ``"gelu"`` (by the error function) or ``"silu"``.  ``p``: from 0 to 1; a multiple of
    2^-32 is what counts, the nearest one, and 1 leaves the residual.  A dropped value is not looked at: NaN and infinity go
    as well.

    ``seed``, ``offset``: whole numbers of 64 bits; the same two drop the same values, whatever the strides, types and device, and two
    calls that are to be independent differ in one of them.  Or ``seed`` is an int64 tensor of two values on the block's device, seed
    and offset, which is read when the kernels run: a captured graph then drops anew with every replay.  It must not change
    between a call and its backward.  Differentiable once, in reverse, with respect to block, residual and bias; without an
    activation nothing of the block is kept for that."""
    on_gpu = block.is_cuda
    if not on_gpu or block.dim() < 1:  # (the native code checks for itself)
        _check(block, residual, bias)
    if activation not in _ACTIVATIONS:
        raise RuntimeError('residual_dropout: activation must be None, "relu", "gelu" or "silu", got %r' % (activation,))
    if isinstance(p, torch.Tensor) or not 0 <= p <= 1:
        raise RuntimeError("residual_dropout: p is a number from 0 to 1, got %r" % (p,))
    seeds = None
    if isinstance(seed, torch.Tensor):
        if tuple(seed.shape) != (2,) or seed.dtype != torch.int64 or not seed.is_contiguous() or offset != 0:
            raise RuntimeError("residual_dropout: a seed on the device is a contiguous int64 tensor of two values, seed and offset")
        seeds, seed = seed, 0
    for name, n in (("seed", seed), ("offset", offset)):
        if isinstance(n, torch.Tensor) or not hasattr(n, "__index__") or not -1 << 63 <= index(n) < 1 << 64:
            raise RuntimeError("residual_dropout: %s must be a whole number of 64 bits, got %r" % (name, n))
    if not on_gpu and any(t is not None and t.device != block.device for t in (residual, bias, seeds)):
        raise RuntimeError("residual_dropout: all tensors must be on one device")
    options = (_ACTIVATIONS[activation], int(round(float(p) * _ALL)), index(seed) & (1 << 64) - 1, index(offset) & (1 << 64) - 1)
    if block.device.type == "cpu":
        return _cpu_dropout(block, residual, bias, seeds, *options)
    if not torch.compiler.is_compiling():
        x = _native.host().residual_dropout_plain(block, residual, bias, seeds, *options)
        if x is not None:
            return x
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (block, residual, bias))
            or torch.jit.is_tracing()):  # (a tracer sees the function)
        return ResidualDropout.apply(block, residual, bias, seeds, options)
    return _native.host().residual_dropout(block, residual, bias, seeds, *options)
