"""The dropout's activations value by value: tails in fp32, NaN and infinity."""
import math

import pytest
import torch

import dropout_words as ref
from fast_transformers_amd.dropout import residual_dropout

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_tails_in_fp32(device, dtype, activation):
    # Each value by itself.  Of gelu's: erfc's argument has two roundings (the factor's and the product's), x (1 + 2^-23), which change
    # erfc(x) by up to 2 x^2 + 1 times as much, z^2 + 1 in half steps of 2^-24 twice; erfc, the products and the result's rounding take sixteen
    # half steps more.  An exponential of z or of z^2 / 2 (two roundings) changes by as many half steps as its argument is large, |z| or z^2.
    z = torch.cat([torch.linspace(-12.5, 9, 4003), torch.tensor([0.0, -0.0, 1e-20, -1e-20, 30.0, -5.0, -5.5, -6.0])]).to(dtype)
    z = torch.cat([z, z[: -len(z) % 8]]).to(device)
    onto = torch.zeros(z.shape, device=device)
    w = z.double().cpu()
    room = (2 * w * w + w.abs() + 18) * 2.0 ** -24
    if activation == "gelu":
        first = 0.5 * torch.special.erfc(-w * math.sqrt(0.5))
        second = w * torch.exp(-0.5 * w * w) / math.sqrt(2 * math.pi)
    else:
        first = 1 / (1 + torch.exp(-w))
        second = w * first / (1 + torch.exp(w))
    leaf = z.clone().requires_grad_(True)
    x = residual_dropout(leaf, onto, p=0.0, seed=1, activation=activation)
    assert ((x.detach().double().cpu() - w * first).abs() <= room * (w * first).abs() + 1e-37).all()
    (grad,) = torch.autograd.grad(x, leaf, torch.ones_like(x))
    slope, half = first + second, torch.finfo(dtype).eps / 2
    # (bf16 slopes' polynomials, 1.6e-7, are three of the half steps)
    assert ((grad.double().cpu() - slope).abs() <= half * slope.abs() + room * (first.abs() + second.abs()) + 1e-37).all()
