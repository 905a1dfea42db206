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


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [24, 21, 5])
def test_nan_that_is_kept_stays_in_the_gradient_of_relu(device, dtype, width):
    """Results of NaN pass the gradient on, as torch's relu does: it is zero where the result is."""
    block = torch.randn(6, width, generator=torch.Generator().manual_seed(1))
    block[2], block[:, 1], block[4, 0], block[4, 2] = float("nan"), float("nan"), float("inf"), -float("inf")
    block = block.to(dtype).to(device).requires_grad_(True)
    bias = torch.zeros(width, device=device, requires_grad=True)
    gx = torch.randn(6, width, generator=torch.Generator().manual_seed(2)).to(dtype).to(device)
    keep = ref.kept(block.numel(), 9, 0, 0.5).view(block.shape).to(device)
    x = residual_dropout(block, p=0.5, seed=9, bias=bias, activation="relu")
    assert torch.equal(torch.isnan(x), torch.isnan(block) & keep)
    wanted = torch.where(keep & ~(block <= 0), 2 * gx, 0.0)
    for leaves in ([block], [block, bias]):
        grads = torch.autograd.grad(x, leaves, gx, retain_graph=True)
        assert torch.equal(grads[0], wanted)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_do_not_look_at_dropped_values(device, dtype, activation):
    gen = torch.Generator().manual_seed(3)
    block, gx = (torch.randn(20, 33, generator=gen).to(dtype).to(device) for _ in range(2))
    bias = torch.randn(33, generator=gen).to(device)
    gone = ~ref.kept(block.numel(), 3, 0, 0.5).view(block.shape).to(device)
    odd = torch.arange(33, device=device) % 2 == 0
    spoiled, spoiled_gx = block.clone(), gx.clone()
    spoiled[gone], spoiled_gx[gone & odd] = float("nan"), float("nan")
    spoiled[gone & odd], spoiled_gx[gone & ~odd] = -float("inf"), float("inf")
    results = []
    for b, g in ((block, gx), (spoiled, spoiled_gx)):
        leaves = [t.clone().requires_grad_(True) for t in (b, bias)]
        x = residual_dropout(leaves[0], p=0.5, seed=3, bias=leaves[1], activation=activation)
        results.append([x.detach(), *torch.autograd.grad(x, leaves, g)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
