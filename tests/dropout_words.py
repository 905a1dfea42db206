"""The dropout behind a block from its definition, a word of 32 bits a value, in whole numbers and 64 bits, for the tests."""
import math

import numpy
import torch

from dropout_reference import BF16, FP32, SUMS, tolerance  # noqa: F401  (of the sums and roundings, which are the same)


def border(p):
    """Words below this are those of dropped values: p 2^32, to the nearest whole number."""
    return round(p * 2 ** 32)


def words(count, seed, offset, start=0):
    """Words start to start + count of Philox4x32-10: word i is word i % 4 of the counter (i // 4, offset)."""
    u32, u64, low = numpy.uint32, numpy.uint64, (1 << 32) - 1
    seed, offset, skip = seed % (1 << 64), offset % (1 << 64), start % 4
    at = numpy.arange(start // 4, (start + count + 3) // 4, dtype=u64)
    c = [at & u64(low), at >> u64(32)] + [numpy.full_like(at, offset >> shift & low) for shift in (0, 32)]
    key = [seed & low, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)  # (both factors below 2^32: no product is cut)
        c = [b >> u64(32) ^ c[1] ^ u64(key[0]), b & u64(low), a >> u64(32) ^ c[3] ^ u64(key[1]), a & u64(low)]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    return numpy.stack(c, -1).reshape(-1)[skip:skip + count].astype(u32)


def kept(count, seed, offset, p, start=0):
    """Which values start to start + count are kept."""
    return torch.from_numpy(words(count, seed, offset, start).astype(numpy.int64) >= border(p))


def dropout(block, residual=None, bias=None, activation=None, keep=None, p=0.0):
    """float64 tensors, differentiable by autograd."""
    z = block if bias is None else block + bias
    if activation == "relu":
        z = torch.relu(z)
    elif activation == "gelu":
        z = z * 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
    elif activation == "silu":
        z = z * torch.sigmoid(z)
    x = torch.where(keep.view(block.shape), z * (1 / (1 - p) if p < 1 else 0.0), torch.zeros_like(z))
    return x if residual is None else x + residual
