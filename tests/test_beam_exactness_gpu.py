"""Attention behind shared pages is off by no more than its inputs' type asks: in bf16 sums as exact as in 32 bits, and the one rounding of
what is stored; in 32 bits scores that lose no more than a sum in a few runs does."""

from __future__ import annotations

import math

import pytest
import torch

from tests.plain import beams as plain
from tests.test_beams_gpu import GROUPS, paged, run_attend

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def check(out, q, k, v, tables, ctx, H, KV, d, scale, sinks=None):
    """A score is off by 2^-24 sqrt(d) of its size, a probability by as much: 2.5e-5 of the sum of |p v| (scores up to 8).  A probability
    goes into its product as two bf16 numbers: the first is off by at most 2^-7 of it (cut), the second by 2^-8 of that, 2^-15.  What
    is stored is off by 2^-8 of itself."""
    want, weight = plain.attend(q, k, v, tables, ctx, H, KV, d, scale, sinks)
    inner = (2.5e-5 + 2.0 ** -15) * weight + 1e-7
    off = (out.cpu().double() - want).abs()
    bound = inner + 2.0 ** -8 * (want.abs() + inner)
    assert bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize("groups", sorted(GROUPS))
@pytest.mark.parametrize("H,KV,d", [(4, 2, 16), (6, 2, 80), (8, 2, 64), (3, 3, 128), (8, 1, 256), (40, 2, 32), (32, 2, 128), (24, 2, 96)])
def test_bf16_outputs_are_rounded_once(groups, H, KV, d):
    k, v, tables, cu, shared, ctx = paged(GROUPS[groups], KV, d, 16, BF16, 15)
    q = (torch.randn(len(ctx), H * d, generator=torch.Generator().manual_seed(11)) * 1.3).to(BF16)
    sinks = torch.randn(H, generator=torch.Generator().manual_seed(2)) if H == 8 else None
    out = run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, d ** -0.5, sinks)
    check(out, q, k, v, tables, ctx, H, KV, d, d ** -0.5, sinks)


@pytest.mark.parametrize("page", [1, 3, 8, 12, 32])
@pytest.mark.parametrize("cuts", [(1, 1), (64, 64)])
def test_bf16_outputs_of_any_pages_and_cuts(page, cuts):
    groups = [(96, [97, 130, 110]), (48, [48, 49]), (0, [200])]
    k, v, tables, cu, shared, ctx = paged(groups, 2, 48, page, BF16, page + 1)
    q = torch.randn(len(ctx), 6 * 48, generator=torch.Generator().manual_seed(page)).to(BF16)
    out = run_attend(q, k, v, tables, cu, shared, ctx, 6, 2, 48, 0.2, cuts=cuts)
    check(out, q, k, v, tables, ctx, 6, 2, 48, 0.2)


@pytest.mark.parametrize("d", [16, 64, 128])
def test_a_value_that_is_infinite_stays_infinite(d):
    """Where a sequence sees it; two of unlike signs are no number, and neither reaches other elements or sequences."""
    H, KV = 4, 2
    k, v, tables, cu, shared, ctx = paged([(64, [70, 90, 66])], KV, d, 16, BF16, 9)
    q = torch.randn(3, H * d, generator=torch.Generator().manual_seed(4)).to(BF16)
    v[tables[0][0], 0, 3, 5] = float("inf")                        # a shared key
    v[tables[0][1], 1, 7, 2] = float("-inf")
    v[tables[0][2], 0, 9, 0], v[tables[0][3], 0, 9, 15] = float("inf"), float("-inf")
    v[tables[1][4], 0, 4, 3] = float("inf")                        # one of the second sequence's own
    out = run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, d ** -0.5).cpu().float().view(3, H, d)
    want, _ = plain.attend(q, k, v, tables, ctx, H, KV, d, d ** -0.5)
    want = want.view(3, H, d)
    assert want[0, 0, 3] == float("inf") and want[1, 3, 7] == float("-inf") and want[2, 1, 9].isnan() and want[1, 0, 4] == float("inf")
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out == float("inf"), want == float("inf"))
    assert torch.equal(out == -float("inf"), want == -float("inf"))


@pytest.mark.parametrize("H,KV", [(1, 1), (20, 2)])
@pytest.mark.parametrize("d", [96, 128, 192, 256])
def test_32_bit_scores_are_summed_in_runs(H, KV, d):
    """A score of 2^11 from one element and a last run of elements whose products are each a quarter of 0.9 half steps of it: added one after
    the other to 2^11 they are lost, four at a time too; summed by themselves first they are there.  Two keys, one with them and one
    without, values 1 and -1: the output is tanh of half their scores' difference.  A score is rounded by half a step (2^-13), and so is
    its product with log2(e) (2^-13 again, ln 2 of it in the exponent), for both keys: 2^-13 (1 + 2 ln 2) of the difference at
    most, half of that in the output, 1.46e-4.  What was lost is 0.9 * n / 4 half steps, n = 32 at least: 4.4e-4."""
    first = {96: 64, 128: 64, 192: 128, 256: 128}[d]
    k, v = torch.zeros(1, KV, 16, d), torch.zeros(1, KV, d, 16)
    k[0, :, :2, 0] = 2.0 ** 11
    k[0, :, 0, first:] = 0.9 * 2.0 ** -15
    v[0, :, :, 0], v[0, :, :, 1] = 1.0, -1.0
    q = torch.zeros(2, H, d)
    q[:, :, 0], q[:, :, first:] = 1.0, 1.0
    for shared in (0, 2):
        out = run_attend(q.view(2, H * d), k, v, [[0], [0]], [0, 2], [shared], [2, 2], H, KV, d, 1.0).cpu().double()
        want, _ = plain.attend(q.view(2, H * d), k, v, [[0], [0]], [2, 2], H, KV, d, 1.0)
        assert bool((out - want).abs().max() <= 2.0 ** -13 * (0.5 + math.log(2.0))), (out[0, 0], want[0, 0])
