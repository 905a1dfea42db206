"""The kernels of the norms around a block against the definition in 64 bits (norm_reference.py, where the tolerances
are derived)."""
import pytest
import torch

import norm_reference as ref
from fast_transformers_amd.norms import residual_norm

pytestmark = pytest.mark.gpu

F, B = torch.float32, torch.bfloat16


@pytest.mark.parametrize("width", [1, 7, 8, 64, 100, 128, 129, 512, 513, 1000, 1024, 1032, 2048, 2056, 4096, 4100, 8192, 8200, 16384])
def test_widths(width):
    if width < 3:  # nothing to normalise
        t = ref.case((37, width), F, B, (37, width), None, None)
        ref.check(ref.both(t, "cuda", None, None, 0.5, "sigmoid"))
        with pytest.raises(RuntimeError, match="at least 3"):
            residual_norm(t["block"].cuda(), after="rms")
        return
    for rows, block, stream in ((1, F, F), (37, B, F), (70, B, B)):
        ref.check(ref.both(ref.case((rows, width), block, stream, (rows, width), "rms", "rms"), "cuda", "rms", "rms", 0.5,
                           "sigmoid"))


@pytest.mark.parametrize("after", [None, "rms", "layer"])
@pytest.mark.parametrize("before", [None, "rms", "layer"])
@pytest.mark.parametrize("stream", [None, F, B])
def test_norms_and_streams(after, before, stream):
    for gate, activation in ((None, None), ((5, 33, 96), "silu"), ((5, 1, 96), "sigmoid"), ((96,), None)):
        for block in (F, B):
            t = ref.case((5, 33, 96), block, stream, gate, after, before, weights=block)
            ref.check(ref.both(t, "cuda", after, before, 0.75, activation))


@pytest.mark.parametrize("gate", [(1, 1, 72), (700, 1, 72), (700, 3, 72), (1, 3, 72), (3, 72)])
def test_shared_gates(gate):
    """One for all rows, one for each of many short runs, full, and one that lies across the rows."""
    ref.check(ref.both(ref.case((700, 3, 72), F, F, gate, "layer", "rms"), "cuda", "layer", "rms", 2.0, "silu"))


def test_many_rows():
    """More rows than the workgroups take at a time, in one segment and in several."""
    for gate in (None, (3, 1, 128), (128,)):
        ref.check(ref.both(ref.case((3, 9001, 128), B, None, gate, "rms", None), "cuda", "rms", None, 1.0, None))


def test_strides_and_alignment():
    gen = torch.Generator().manual_seed(9)
    wide = torch.randn(6, 11, 3 * 64, generator=gen)
    want = ref.residual_norm(wide[..., 64:128].double(), wide[..., 128:].double(), wide[..., :64].double(),
                             ("rms",), ("layer",), 1.0, "silu")
    dev = wide.cuda()
    x, h = residual_norm(dev[..., 64:128], dev[..., 128:], dev[..., :64], after=("rms",), before=("layer",), activation="silu")
    assert ref.far(x, want[0]) <= ref.FP32 and ref.far(h, want[1]) <= ref.FP32
    odd = dev.flatten()[1:1 + 65 * 190].view(65, 190)[:, 3:131]            # 4-byte boundaries
    x, h = residual_norm(odd, before="rms")
    want = ref.residual_norm(odd.double().cpu(), None, None, None, ("rms",), 1.0, None)
    assert ref.far(x, want[0]) <= ref.FP32 and ref.far(h, want[1]) <= ref.FP32
    turned = dev.permute(1, 0, 2)                                          # two row strides
    x, h = residual_norm(turned, turned, after="layer")
    want = ref.residual_norm(turned.double().cpu(), turned.double().cpu(), None, ("layer",), None, 1.0, None)
    assert ref.far(x, want[0]) <= ref.FP32 and h is None


def test_one_result_used_and_single_gradients():
    t = ref.case((4, 40, 64), F, F, (4, 1, 64), "rms", "layer")
    dev = {n: x.cuda().requires_grad_(True) for n, x in t.items()}
    wide = {n: x.double().requires_grad_(True) for n, x in t.items()}
    args = lambda d: dict(after=ref.spec(d, "a", "rms"), before=ref.spec(d, "b", "layer"))  # noqa: E731
    for pick in (0, 1):
        got = residual_norm(dev["block"], dev["residual"], dev["gate"], **args(dev))[pick]
        want = ref.residual_norm(wide["block"], wide["residual"], wide["gate"], ref.spec(wide, "a", "rms"),
                                 ref.spec(wide, "b", "layer"), 1.0, None)[pick]
        for n in t:
            a = torch.autograd.grad(got.square().sum(), dev[n], retain_graph=True, allow_unused=True)[0]
            b = torch.autograd.grad(want.square().sum(), wide[n], retain_graph=True, allow_unused=True)[0]
            if b is None:
                assert a is None or not a.any()
            else:
                assert ref.far(a, b) <= ref.FP32, (pick, n)


def test_rows_of_zeros_large_means_and_no_rows():
    x, h = residual_norm(torch.zeros(3, 64, device="cuda"), after="layer", before="rms")
    assert not x.any() and not h.any()
    # the variance is that of the values, not of their squares: means of 1000 deviations leave 14 bits of it
    r = torch.randn(50, 512, generator=torch.Generator().manual_seed(1)) + 1000.0
    x, _ = residual_norm(r.cuda(), after="layer")
    want, _ = ref.residual_norm(r.double(), None, None, ("layer",), None, 1.0, None)
    # (the mean is off by a few half steps of 2^-24 x 1000: 1000 x 2^-24 x 4 of a deviation)
    assert ref.far(x, want) <= 1000 * 2.0 ** -24 * 4
    block = torch.zeros(0, 5, 16, device="cuda", requires_grad=True)
    weight = torch.ones(16, device="cuda", requires_grad=True)
    x, h = residual_norm(block, gate=torch.ones(16, device="cuda"), before=("rms", weight))
    (x.sum() + h.sum()).backward()
    assert x.shape == h.shape == block.shape and not weight.grad.any() and block.grad.shape == block.shape


def test_results_do_not_depend_on_the_order_of_atomics():
    t = {n: x.cuda().requires_grad_(True) for n, x in ref.case((8, 500, 512), B, F, (8, 1, 512), "layer", "layer").items()}

    def once():
        x, h = residual_norm(t["block"], t["residual"], t["gate"], after=ref.spec(t, "a", "layer"),
                             before=ref.spec(t, "b", "layer"))
        return [x, h, *torch.autograd.grad([x, h], list(t.values()), [torch.ones_like(x), torch.ones_like(h)])]
    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)
