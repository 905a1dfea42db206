"""Decayed linear attention of many chains, whose workgroups go through all segments of one: types, decays, widths, slices, shared
key heads, and sequences that end in any of the segments, against the definition in 64 bits."""
import pytest
import torch

import decay_reference as ref
from fast_transformers_amd import _native
from test_decayed_attention_gpu import check, results

pytestmark = pytest.mark.gpu

# (some have two segments, some three; H on as many key heads or fewer)
SIZES = [(128, 4, 2, 2100, 64, 64), (60, 4, 2, 2100, 24, 136), (60, 4, 4, 2100, 72, 128), (60, 4, 1, 2100, 128, 19), (32, 16, 16, 1100, 8, 8)]


@pytest.mark.parametrize("decay", ["position", "head"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_segments_one_after_the_other(sizes, dtype, decay):
    N, H, Hk, L, E, M = sizes
    plan = _native.decayed_plan(*sizes, _native.FTC_BF16 if dtype == torch.bfloat16 else _native.FTC_F32)
    assert "one after the other" in plan
    segments, length = int(plan.split()[1]), int(plan.split()[3].rstrip(","))
    # a few sequences' own values, those of the first of them for all others, whose results' gradients are zero
    some = [0, 1, 2, N // 2, N - 2, N - 1]
    ends = [L, 0, length - 1, length + 70, (segments - 1) * length, L - 1]
    few = ref.inputs(len(some), H, Hk, L, E, M, dtype=dtype, decay=decay, device="cuda")
    if decay == "head":
        few[3] /= 16                       # (memories of hundreds of positions: across the segments)
    gen = torch.Generator(device="cuda").manual_seed(1)
    few_go = torch.randn(few[2].shape, generator=gen, device="cuda").to(dtype)
    few_gs = torch.randn(few[4].shape, generator=gen, device="cuda")

    def spread(t, rest):
        every = (t[:1] if rest else torch.zeros_like(t[:1])).expand(N, *t.shape[1:]).clone(memory_format=torch.contiguous_format)
        every[some] = t
        return every
    args = [t if t.dim() == 1 else spread(t, True) for t in few]
    go, gs = spread(few_go, False), spread(few_gs, False)
    lengths = torch.full((N,), L, device="cuda")
    lengths[some] = torch.tensor(ends, device="cuda")
    wide = [t.double().requires_grad_(True) for t in few]
    for lens, few_lens in ((None, None), (lengths, lengths[some])):
        got = results(args, go, gs, lengths=lens)
        want = ref.attention(*wide, scale=E ** -0.5, lengths=few_lens)
        want = [*want, *torch.autograd.grad(want, wide, [few_go.double(), few_gs.double()])]
        check([t if t.dim() == 1 else t[some] for t in got], want)
        if lens is not None:
            for i, end in zip(some, ends):
                assert not got[0][i, :, end:].any() and not got[4][i, :, end:].any() and not got[2][i, :, end:].any()
