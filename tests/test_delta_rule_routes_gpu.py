"""The gated delta rule on every route of its scans: wavefronts alone, in pairs and in fours, in one launch and in
segments, with and without wide accesses, on groups that are not full, with ragged lengths.  Each case names the route
that it is there for, and fails if the call takes another.  Against the definition in 64 bits, position by position on
the GPU (tolerances: delta_reference.py)."""
import pytest
import torch

import delta_reference as ref
from fast_transformers_amd import _native
from fast_transformers_amd.delta_rule import gated_delta_rule

F, B = torch.float32, torch.bfloat16

# route, type, N, H, Hk, L, E, M (16 columns of values to a wavefront; wide accesses where E and M are multiples of 8)
CASES = [
    ("scan 1", F, 1, 6, 3, 130, 64, 48),
    ("scan 1", B, 2, 9, 9, 130, 100, 45),
    ("scan 2", F, 4, 16, 8, 150, 64, 96),
    ("scan 2", F, 4, 16, 16, 130, 37, 90),
    ("scan 2", B, 4, 16, 8, 150, 64, 96),
    ("scan 2", B, 4, 16, 16, 130, 37, 90),
    ("scan 2", B, 4, 16, 8, 150, 128, 96),
    ("scan 2", B, 4, 16, 4, 130, 100, 90),
    ("scan 4", F, 8, 15, 5, 150, 64, 80),
    ("scan 4", F, 8, 15, 15, 130, 33, 77),
    ("scan 4", F, 3, 5, 5, 130, 128, 80),
    ("scan 4", F, 8, 15, 3, 130, 101, 77),
    ("scan 4", B, 8, 15, 5, 150, 64, 80),
    ("scan 4", B, 8, 15, 15, 130, 33, 77),
    ("scan 4", B, 8, 15, 5, 130, 128, 80),
    ("scan 4", B, 8, 15, 3, 130, 101, 77),
    ("segments 5, maps 2, scan 1", F, 4, 16, 8, 1593, 16, 16),
    ("segments 5, maps 2, scan 1", B, 4, 16, 8, 1593, 16, 16),
    ("segments 6, maps 4, scan 1", F, 4, 16, 16, 2290, 11, 13),
    ("segments 6, maps 4, scan 1", B, 4, 16, 16, 2290, 11, 13),
    ("segments 6, maps 4, scan 2", F, 2, 16, 8, 2290, 32, 32),
    ("segments 6, maps 4, scan 2", B, 2, 16, 8, 2290, 29, 27),
    ("segments 4, maps 4, scan 4", F, 2, 8, 4, 1020, 72, 40),
    ("segments 4, maps 2, scan 1", B, 2, 8, 4, 2040, 128, 32),
    ("segments 4, maps 4, scan 1", B, 2, 8, 8, 2040, 117, 37),
]


def ids(case):
    return "%s-%s-%s" % (case[0].replace(", ", "_").replace(" ", ""), "bf16" if case[1] == B else "fp32", "x".join(map(str, case[2:])))


def plan(case, keep=True):
    return _native.delta_plan(*case[2:], _native.FTC_F32 if case[1] == F else _native.FTC_BF16, keep)


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_cases_take_their_routes(case):
    expected = "chunks %d, %s" % ((case[5] + 63) // 64, case[0])
    assert plan(case) == expected and plan(case, keep=False) == expected


def test_every_route_has_a_case():
    """Wavefronts that share, by type and width of the keys, in each launch."""
    seen = set()
    for case in CASES:
        words = case[0].replace(",", "").split()
        for launch, by in zip(words[::2], words[1::2]):
            if launch != "segments":
                seen.add((launch, int(by), case[1], case[6] > 64))
    for dtype in (F, B):
        for wide in (False, True):
            alone = not (dtype == F and wide)   # (three pieces of 128 key columns: always in fours)
            for by in (1, 2, 4) if alone else (4,):
                assert ("scan", by, dtype, wide) in seen
            # (maps by one wavefront: the long chains of test_delta_rule_use_gpu)
            for by in (2, 4) if alone else (4,):
                assert ("maps", by, dtype, wide) in seen


def test_plans():
    assert _native.delta_plan(1, 1, 1, 8, 64, 64, keep=False) == "steps"
    assert _native.delta_plan(1, 1, 1, 8, 64, 64) == "chunks 1, scan 1"
    assert _native.delta_plan(1, 1, 1, 0, 64, 64) == "steps"
    assert _native.delta_plan(0, 1, 1, 9, 64, 64) == ""
    assert _native.delta_plan(1, 2, 1, 1000, 64, 64) == "chunks 16, segments 4, maps 1, scan 1"
    for bad in ((1, 3, 2, 9, 8, 8), (1, 1, 1, 9, 129, 8), (1, 1, 1, 9, 8, 513), (-1, 1, 1, 9, 8, 8)):
        with pytest.raises(RuntimeError):
            _native.delta_plan(*bad)
    with pytest.raises(RuntimeError, match="dtype"):
        _native.delta_plan(1, 1, 1, 9, 8, 8, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
@pytest.mark.parametrize("case", CASES, ids=ids)
def test_routes_follow_the_definition(case, ragged):
    route, dtype, N, H, Hk, L, E, M = case
    args = ref.inputs(N, H, Hk, L, E, M, dtype=dtype, device="cuda", seed=L + E + M)
    args[3][:, :1].mul_(0.02)                                            # (a head that remembers over segments)
    lengths = None
    if ragged:
        ends = [L, 0, 1, 64, L // 2, 65, L - 1, L // 3]
        lengths = torch.tensor((ends if N > 1 else ends[4:])[:N], device="cuda")
    gen = torch.Generator().manual_seed(5)
    go = torch.randn(args[2].shape, generator=gen).to(dtype).cuda()
    gs = 0.3 * torch.randn(args[5].shape, generator=gen).cuda()
    leaves = [t.detach().requires_grad_(True) for t in args]
    out, state = gated_delta_rule(*leaves, normalize=True, lengths=lengths, return_state=True)
    got = [out.detach(), state.detach(), *torch.autograd.grad([out, state], leaves, [go, gs])]
    torch.cuda.synchronize()
    wide = [t.detach().double().requires_grad_(True) for t in args]
    want, want_state = ref.rule(*wide, scale=E ** -0.5, normalize=True, lengths=lengths)
    want = [want, want_state, *torch.autograd.grad([want, want_state], wide, [go.double(), gs.double()])]
    errors = [ref.far(a, b) for a, b in zip(got, want)]
    print(["%.2g" % e for e in errors], flush=True)
    for a, e in zip(got, errors):
        assert e <= ref.tolerance(a.dtype), errors
    with torch.no_grad():                                                # (nothing kept: the same values)
        out, state = gated_delta_rule(*args, normalize=True, lengths=lengths, return_state=True)
    assert torch.equal(out, got[0]) and torch.equal(state, got[1])
