# SPDX-License-Identifier: MIT
"""Attention on the GPU where few bits of a probability matter: long caches of which
one key has most of a row's weight."""

import math

import pytest
import torch

import beamgrad_amd as bg

pytestmark = pytest.mark.gpu

HALF_STEP = 2.0**-11  # of float16


@pytest.mark.parametrize("ahead", [12, 16, 17, 18, 20])
@pytest.mark.parametrize("N, H, Hkv", [(1, 1, 1), (1, 16, 1), (40, 1, 1), (128, 1, 1), (300, 1, 1), (1024, 64, 64)])
def test_many_small_probabilities_beside_a_large_one(N, H, Hkv, ahead):
    """The first key's score is `ahead`, 131000 others' are 0: their sum counts. The
    values are 0 and 1, so the result is the others' share of the weight. Of many
    rows and heads, one wavefront meets all keys of a row."""
    L, D, page = 131000, 64, 128
    pages = -(-L // page)
    k = torch.zeros(pages, page, 1, D, dtype=torch.float16, device="cuda")
    v = torch.ones_like(k)
    k[0, 0, 0, 0], v[0, 0] = ahead, 0
    q = torch.zeros(1, N, H, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0  # whose product with the scale of 1/8 is 1
    table = bg.PageTable(torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.tensor([L], dtype=torch.int32, device="cuda"),
                         torch.ones(pages, dtype=torch.int32, device="cuda"))
    k, v = (t.expand(pages, page, Hkv, D) for t in (k, v))
    out, lse = bg.tree_attention(q, k, v, table, return_lse=True)
    others = (L - N + torch.arange(N, dtype=torch.float64)) * math.exp(-ahead)  # token i sees L - N + i keys beside the first
    want = (others / (1 + others))[None, :, None, None]
    # The scores are exact. A probability relative to its row's largest of 1 or more,
    # 2^7 times that where it is rounded: half a step of it, or half the least step,
    # 2^-25; the result's own rounding; float32 sums and exponentials.
    bound = 2 * HALF_STEP * want + L * 2.0**-25 * 2.0**-7 + (2 * L + 64) * 2.0**-24 * want
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by {(off / want).max():.3g} of the result, {(off / bound).max():.3g} of its bound"
    want = ahead + torch.log1p(others)[None, :, None]
    # the sums round by 2^-24 of themselves a step, the first key's weight in them
    assert bool(((lse.cpu().double() - want).abs() <= (2 * L + 64) * 2.0**-24 + 2.0**-20 + 2.0**-22 * want).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_large_scores_stay_finite(dtype):
    """Scores up to 10^6 that rise along the keys: the probabilities that are rounded
    stay in their type's range."""
    L, N, D = 900, 128, 64
    k = torch.zeros(15, 64, 1, D, dtype=dtype, device="cuda")
    k.view(960, D)[:, 0] = (torch.arange(960, device="cuda") * 64).to(dtype)
    q = torch.zeros(1, N, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = 128.0
    v = torch.randn(15, 64, 1, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(dtype)
    table = bg.PageTable(torch.arange(15, dtype=torch.int32, device="cuda")[None], torch.tensor([L], dtype=torch.int32, device="cuda"),
                         torch.ones(15, dtype=torch.int32, device="cuda"))
    out = bg.tree_attention(q, k, v, table)
    scores = k.view(960, D)[:, 0].double() * 16
    for i in range(0, N, 13):
        seen = L - N + i + 1
        p = torch.softmax(scores[:seen], 0)
        want = p @ v.view(960, D)[:seen].double()
        half = torch.finfo(dtype).eps / 2
        # scores are exact products; their multiples of log2(e), of up to 2^21, round by
        # 2^-4 in the exponent twice, which moves each weight's logarithm by as much
        grow = math.expm1(2 * 2 * 2.0**-4 * math.log(2))
        bound = half * want.abs() + (half + grow + 1e-4) * (p @ v.view(960, D)[:seen].double().abs()) * (1 + half) + 2.0**-20
        assert bool(((out[0, i, 0].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [1e-38, 1e-45])
def test_the_smallest_scales(dtype, scale):
    """All scores are 0: each row is the mean of what it sees, also where the first
    keys are another row's alone. So many heads that none is cut."""
    N, H, D, page = 100, 1024, 64, 16
    parents = torch.full((1, N), -1, dtype=torch.int32)
    parents[0, 96], parents[0, 98] = 5, 70
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(1, N, H, D, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(7, page, 1, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    table = bg.PageTable(torch.arange(7, dtype=torch.int32, device="cuda")[None], torch.tensor([N], dtype=torch.int32, device="cuda"),
                         torch.ones(7, dtype=torch.int32, device="cuda"))
    out, lse = bg.tree_attention(q, k.expand(7, page, H, D), v.expand(7, page, H, D), table, parents=parents.cuda(), scale=scale,
                                 return_lse=True)
    values = v.view(7 * page, D).double()
    for i in range(N):
        seen = [i] + [int(parents[0, i])] * int(parents[0, i] >= 0)
        want = values[seen].mean(0)
        # sums of one or two terms, and the rounding of the result
        assert bool(((out[0, i].double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0**-20) * values[seen].abs().sum(0)).all())
        assert bool(((lse[0, i] - math.log(len(seen))).abs() <= 2.0**-20).all())
