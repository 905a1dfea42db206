"""The norms around a block on the CPU: the implementation for CPU tensors against the definition, and refusals."""
import ctypes

import pytest
import torch

import norm_reference as ref
from fast_transformers_amd import _native
from fast_transformers_amd.norms import residual_norm


@pytest.mark.parametrize("after", [None, "rms", "layer"])
@pytest.mark.parametrize("before", [None, "rms", "layer"])
@pytest.mark.parametrize("gate", [None, (3, 5, 24), (3, 1, 24), (24,), (1, 5, 1, 24)])
def test_cpu_tensors_follow_the_definition(after, before, gate):
    shape = (3, 5, 24) if gate is None or len(gate) < 4 else (3, 5, 2, 24)
    for activation in (None, "sigmoid", "silu"):
        t = ref.case(shape, torch.float32, torch.float32, gate, after, before)
        ref.check(ref.both(t, "cpu", after, before, 0.5, activation))


def _refused(match, block=torch.zeros(2, 3, 8), *args, **options):
    with pytest.raises(RuntimeError, match=match):
        residual_norm(block, *args, **options)


def test_refusals():
    x = torch.zeros(2, 3, 8)
    _refused("1 to 16384", torch.zeros(2, 0))
    _refused("1 to 16384", torch.zeros(2, 16385))
    _refused("1 to 16384", torch.tensor(1.0))
    _refused("at least 3", x[..., :1], after="rms")
    _refused("at least 3", x[..., :2], before="layer")
    _refused("float32 or bfloat16", x.half())
    _refused("residual must be", x, x.double())
    _refused("the residual has shape", x, x[:, :2])
    _refused("does not fit", x, None, torch.zeros(2, 2, 8))
    _refused("does not fit", x, None, torch.zeros(2, 3, 1))
    _refused("does not fit", x, None, torch.zeros(1, 2, 3, 8))
    _refused("activation", x, None, x, activation="relu")
    _refused("after must be", x, after=("batch",))
    _refused("before must be", x, before=())
    _refused("vectors of 8", x, before=("rms", torch.zeros(7)))
    _refused("vectors of 8", x, after=("layer", torch.zeros(8), torch.zeros(8).half()))


def test_c_abi_refuses_on_the_host():
    lib = _native.load()

    def call(x=256, h=None, stats=None, **change):
        c = _native.ResidualNormCall()
        c.block = _native.Rows(256, 8, 0)
        c.rows, c.width, c.scale, c.eps = 4, 8, 1.0, 1e-6
        for n, v in change.items():
            setattr(c, n, v)
        xr, hr = _native.Rows(x, 8, 0), _native.Rows(h, 8, 0)
        return lib.ftc_residual_norm(ctypes.byref(c), ctypes.byref(xr), ctypes.byref(hr), stats, None)
    assert lib.ftc_residual_norm(None, None, None, None, None) == -1
    assert call(rows=-1) == -1
    assert call(width=0) == -2 and call(width=16385) == -2
    assert call(width=2, after=_native.Norm(None, None, 1, 0, 0)) == -2
    assert call(activation=3) == -1
    assert call(block=_native.Rows(256, 8, 2)) == -1 and call(block=_native.Rows(None, 8, 0)) == -1
    assert call(after=_native.Norm(None, None, 3, 0, 0)) == -1
    assert call(gate=_native.Rows(256, 8, 0), gate_rows=3) == -1
    assert call(gate=_native.Rows(256, 8, 0), gate_rows=0) == -1
    assert call(x=None) == -1
    assert call(before=_native.Norm(None, None, 1, 0, 0)) == -1      # no h
    assert call(h=256) == -1                                         # no norm that makes it
    c = _native.ResidualNormCall()
    c.block, c.after = _native.Rows(256, 8, 0), _native.Norm(256, None, 1, 0, 0)
    c.rows, c.width = 4, 8
    assert lib.ftc_residual_norm_backward_workspace_bytes(ctypes.byref(c)) > 0
    none = [None] * 5
    assert lib.ftc_residual_norm_backward(ctypes.byref(c), None, *none, None, None, None, None, None, 0, None) == -1
    assert lib.ftc_residual_norm_backward(ctypes.byref(c), 256, *none, None, None, None, None, None, 0, None) == -3
