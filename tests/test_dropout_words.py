"""What the dropout behind a block keeps: a word of 32 bits a value against p 2^32.  Results and gradients against the
definition in 64 bits, over widths, types, layouts, shares next to nothing and to one, and the layers that call it."""
import ctypes
import types

import numpy
import pytest
import torch

import dropout_reference as published
import dropout_words as ref
import test_decayed_layers as layers
from delta_reference import far
from fast_transformers_amd import _native
from fast_transformers_amd.dropout import ResidualDropout, residual_dropout

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
SEED, OFFSET = (1 << 63) + 987654321, (1 << 35) + 11


def test_the_oracle_has_the_published_words():
    low = (1 << 32) - 1
    for seed, offset, start in ((0, 0, 0), (SEED, OFFSET, 0), (12345, (1 << 64) - 1, (1 << 36) - 5), (-1, 7, 2)):
        want = [published.words((i // 4 & low, i // 4 >> 32, offset & low, offset >> 32), (seed & low, seed >> 32 & low))[i % 4]
                for i in range(start, start + 11)]
        assert ref.words(11, seed, offset, start).tolist() == want


def inputs(device, shape, dtype, stream, bias):
    gen = torch.Generator().manual_seed(5)
    draw = lambda s, d: torch.randn(s, generator=gen).to(d).to(device)  # noqa: E731
    block = draw(shape, dtype)
    residual = None if stream is None else draw(shape, stream)
    return block, residual, None if bias is None else draw(shape[-1:], bias), draw(shape, stream or dtype)


def check(device, shape, dtype, stream, bias_type, activation, p, seed=SEED, offset=OFFSET):
    block, residual, bias, gx = inputs(device, shape, dtype, stream, bias_type)
    leaves = [t.requires_grad_(True) for t in (block, residual, bias) if t is not None]
    x = residual_dropout(block, residual, p=p, seed=seed, offset=offset, bias=bias, activation=activation)
    keep = ref.kept(block.numel(), seed, offset, p)
    wide = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    want = ref.dropout(wide[0], None if stream is None else wide[1], None if bias is None else wide[-1], activation, keep, p)
    got, wanted = torch.autograd.grad(x, leaves, gx), torch.autograd.grad(want, wide, gx.double().cpu())
    errors = [far(x, want)] + [far(a, b) for a, b in zip(got, wanted)]
    print(["%.2g" % e for e in errors], flush=True)
    assert x.dtype == (stream or dtype) and errors[0] <= ref.tolerance(x.dtype)
    for t, a, e in zip(leaves, got, errors[1:]):
        assert a.dtype == t.dtype and e <= ref.tolerance(a.dtype) + (ref.SUMS if t is bias else 0)
    # what was dropped is the residual, or nothing, to the last bit
    gone = ~keep.view(shape).to(device)
    assert torch.equal(x.detach()[gone], torch.zeros_like(x.detach())[gone] if residual is None else residual.detach()[gone])
    assert not got[0][gone].any()
    with torch.no_grad():
        assert torch.equal(x, residual_dropout(block, residual, p=p, seed=seed, offset=offset, bias=bias, activation=activation))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 8, 9, 10, 12, 15, 16, 20, 31, 64, 100, 257, 1000, 2056, 2060])
@pytest.mark.parametrize("dtype, stream", [(torch.float32, None), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.bfloat16, torch.bfloat16), (torch.bfloat16, None)])
def test_widths(device, width, dtype, stream):
    check(device, (3, 5, width), dtype, stream, torch.float32, "relu", 0.3)
    check(device, (11, width), dtype, stream, None, None, 0.3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_activations(device, dtype, bias, activation):
    for shape in ((40, 64), (37, 43), (37, 44)):
        check(device, shape, dtype, None, bias, activation, 0.3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("p", [0.0, 2.0 ** -32, 0.001, 0.1, 0.5, 0.999, 1.0])
def test_shares(device, p):
    for width in (50, 48):
        check(device, (9, width), torch.float32, torch.float32, torch.float32, "gelu", p)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows, width", [(5000, 24), (700, 333), (3, 20001), (1, 1), (1, 100000)])
def test_many_rows_and_wide_ones(device, rows, width):
    check(device, (rows, width), torch.bfloat16, torch.float32, torch.float32, "silu", 0.1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("p", [1e-5, 7e-6, 0.999995])
def test_shares_next_to_the_ends(device, p):
    """Each of them is a share of its own: what is dropped is what the words say, and the factor belongs to it."""
    for shape in ((1 << 10, 1 << 10), (1000, 1001)):
        keep = ref.kept(shape[0] * shape[1], 3, 0, p).view(shape)
        few = min(int((~keep).sum()), int(keep.sum()))
        assert 0 < few < 40                                    # (some are dropped, or some kept: the case says something)
        x = residual_dropout(torch.ones(shape, device=device), p=p, seed=3).cpu()
        assert torch.equal(x != 0, keep)
        # (p is the multiple of 2^-32 next to it, off by 2^-33 at most; two roundings)
        assert ((x[keep].double() * (1 - p) - 1).abs() <= 2.0 ** -33 / (1 - p) + 2.0 ** -23).all()


@pytest.mark.parametrize("device", DEVICES)
def test_a_share_between_two_words(device):
    """A value is kept where its word is p 2^32 or more, to the last bit of it."""
    seed, offset, width = 77, 5, 64
    words = ref.words(width, seed, offset).astype(numpy.int64)
    ones = torch.ones(1, width, device=device)
    for i in (0, 1, 5, 63, int(words.argmin()), int(words.argmax())):
        for by in (-1, 0, 1):
            p = (int(words[i]) + by) / 2 ** 32
            x = residual_dropout(ones, p=p, seed=seed, offset=offset)[0].cpu()
            assert (x[i] != 0) == (by <= 0)
            assert torch.equal(x != 0, torch.from_numpy(words >= int(words[i]) + by))


@pytest.mark.parametrize("device", DEVICES)
def test_dropped_values_may_be_anything(device):
    for dtype in (torch.float32, torch.bfloat16):
        block, residual, bias, gx = inputs(device, (20, 33), dtype, dtype, torch.float32)
        gone = ~ref.kept(block.numel(), 3, 0, 0.5).view(block.shape).to(device)
        spoiled = block.clone()
        spoiled[gone] = float("nan")
        spoiled[gone & (torch.arange(33, device=device) % 2 == 0)] = float("inf")
        results = []
        for b in (block, spoiled):
            leaves = [t.clone().requires_grad_(True) for t in (b, residual, bias)]
            x = residual_dropout(leaves[0], leaves[1], p=0.5, seed=3, bias=leaves[2], activation="relu")
            results.append([x.detach(), *torch.autograd.grad(x, leaves, gx)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        everything = torch.full_like(block, float("nan"))
        assert torch.equal(residual_dropout(everything, residual, p=1, seed=3, bias=bias, activation="gelu"), residual)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1 << 18, (1 << 18) - 3])
def test_far_values_count_beyond_32_bits(width):
    """Values behind the first 2^32 and 2^34 have counters of their own."""
    for rows, seed in (((1 << 14) + 2, 5), ((1 << 16) + 2, 6)):
        x = torch.ones(1, width, device="cuda", dtype=torch.bfloat16).expand(rows, width)
        out = residual_dropout(x, p=0.5, seed=seed)
        for row in (rows - 1, rows - 2):
            assert torch.equal(out[row].cpu() != 0, ref.kept(width, seed, 0, 0.5, start=row * width))


@pytest.mark.gpu
def test_both_engines_have_one_option():
    block, residual, bias, gx = inputs("cuda", (6, 40), torch.bfloat16, torch.float32, torch.float32)
    for p in (0.2, 0.0, 1.0):
        plain = residual_dropout(block, residual, p=p, seed=8, bias=bias, activation="silu")
        assert torch.equal(plain, ResidualDropout.apply(block, residual, bias, None, (3, ref.border(p), 8, 0)))


def test_refusals_of_the_library():
    lib = _native.load()
    rows = _native.Rows(256, 8, 0)
    good = dict(block=rows, residual=_native.Rows(), rows=0, width=8, activation=0)
    for dropped, rest, status in ((0, 0, 0), (10, 65535, 0), (65535, 65535, 0), (65536, 0, 0), (65536, 1, -1), (65537, 0, -1), (3, 65536, -1)):
        call = _native.ResidualDropoutCall(**good, dropped=dropped, dropped_rest=rest)
        assert lib.ftc_residual_dropout(ctypes.byref(call), ctypes.byref(rows), None) == status, (dropped, rest)
        assert status == 0 or "dropped" in _native.last_error()


@pytest.fixture
def defined(monkeypatch):
    """The layers' definition (tests/test_decayed_layers.py) with what words drop; its shares are parts of 65536."""
    monkeypatch.setattr(layers, "drop", types.SimpleNamespace(
        kept=lambda count, seed, offset, dropped: ref.kept(count, seed, offset, dropped / 65536),
        dropout=lambda block, residual, bias, activation, keep, dropped: ref.dropout(block, residual, bias, activation, keep, dropped / 65536)))


@pytest.mark.parametrize("kind, activation", [("position", "gelu"), ("head", "silu")])
@pytest.mark.parametrize("device", DEVICES)
def test_training_follows_the_definitions(defined, device, kind, activation):
    layers.test_training_follows_the_definitions(device, kind, activation)


@pytest.mark.parametrize("device", DEVICES)
def test_what_is_dropped(defined, device):
    layers.test_what_is_dropped(device)


@pytest.mark.parametrize("device", DEVICES)
def test_half_precision_model(defined, device, monkeypatch):
    # (a share that is a whole number of parts of 65536)
    made = layers.model
    monkeypatch.setattr(layers, "model", lambda *args, **kwargs: made(*args, **{**kwargs, "dropout": 0.125}))
    layers.test_half_precision_model_keeps_its_stream_in_fp32(device)
