"""The operators of beam search against the plain 64-bit implementation, at the sizes, masks, layouts and orders where
they can go wrong, and a run of all three."""

from __future__ import annotations

import math
import random

import pytest
import torch

from tests.plain import beams as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def ops():
    from kvforge_amd.kernels import ops as o
    return o


# ------------------------------------------------------------------------------------- selection
def run_select(logits, scores, cu, count, outs=None, work=None):
    o = ops()
    r = len(cu) - 1
    outs = outs or (torch.full((r, count), 7.0, device=DEV), torch.full((r, count), 7, dtype=torch.int32, device=DEV),
                    torch.full((r, count), 7, dtype=torch.int32, device=DEV))
    work = work or o.beam_select_workspace(logits.shape[0], logits.shape[1], count, DEV)
    o.beam_select(logits, scores, torch.tensor(cu, dtype=torch.int32, device=DEV), *outs, work)
    return outs


def check_select(logits, scores, cu, count, outs):
    """A score is off by its rounding to 32 bits, 2^-24 of it, and by the sum's error: every exponential is off by a few 2^-24
    of itself (the hardware's, one unit in the last place, and two roundings ahead of it), the sum and so its logarithm by as much: 2^-21."""
    want = plain.select(logits, scores, cu, count + 1)
    total = plain.candidate_scores(logits, scores)
    got_s, got_b, got_t = (t.cpu() for t in outs)
    for r, expected in enumerate(want):
        n = min(count, len(expected))
        assert got_b[r, n:].eq(-1).all() and got_t[r, n:].eq(-1).all() and got_s[r, n:].eq(-math.inf).all()
        seen = set()
        for i in range(n):
            s, b, t = expected[i]
            gb, gt = int(got_b[r, i]), int(got_t[r, i])
            assert abs(float(got_s[r, i]) - s) <= 2.0 ** -24 * abs(s) + 2.0 ** -21, (r, i, s)
            assert (gb, gt) not in seen and 0 <= gb < cu[r + 1] - cu[r]
            seen.add((gb, gt))
            # scores nearer than the sums' error may change places across beams; equal ones of a beam may not
            near = [x for x in expected if abs(x[0] - s) <= 2.0 ** -20 and x[1] != b]
            if not near:
                assert (gb, gt) == (b, t), (r, i, expected[i], (gb, gt))
            else:
                assert abs(float(total[cu[r] + gb, gt]) - s) <= 2.0 ** -20


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,beams,count", [
    (1, 1, 1, 1), (1, 5, 1, 8), (4, 8192, 4, 8), (3, 2049, 3, 6), (7, 50001, 7, 14), (6, 2047, 2, 4), (24, 9001, 12, 24),
    (32, 1000, 16, 32), (5, 300, 5, 64), (64, 8193, 32, 64), (40, 128256, 8, 16), (2, 65, 1, 64), (66, 128256, 6, 12)])
def test_selection(dtype, rows, vocab, beams, count):
    g = torch.Generator().manual_seed(rows * vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).to(DEV)
    scores = (-torch.rand(rows, generator=g) * 5).to(DEV)
    cu = list(range(0, rows + 1, beams))
    check_select(logits, scores, cu, count, run_select(logits, scores, cu, count))


def test_selection_of_beams_of_their_own_number_dead_ones_and_none():
    g = torch.Generator().manual_seed(3)
    cu = [0, 3, 3, 4, 12, 14, 14]
    logits = (torch.randn(14, 4099, generator=g) * 2)
    scores = -torch.rand(14, generator=g) * 4
    for row, s in ((1, -math.inf), (3, math.nan), (5, math.inf), (12, -math.inf), (13, -math.inf)):
        scores[row] = s
    logits[1] = math.nan          # unread
    logits, scores = logits.to(DEV), scores.to(DEV)
    outs = run_select(logits, scores, cu, 10)
    check_select(logits, scores, cu, 10, outs)
    assert outs[1][[1, 2, 4, 5]].eq(-1).all()


@pytest.mark.parametrize("rows,cu,vocab,count", [(150, [0, 70, 71, 150], 900, 20), (300, [0, 300], 70, 64), (64, [0, 64], 9000, 32)])
def test_selection_of_more_beams_than_are_merged_at_a_time(rows, cu, vocab, count):
    g = torch.Generator().manual_seed(rows)
    logits = (torch.randn(rows, vocab, generator=g) * 2).to(DEV)
    scores = (-torch.rand(rows, generator=g) * 3).to(DEV)
    check_select(logits, scores, cu, count, run_select(logits, scores, cu, count))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [70, 2500, 20000])
def test_selection_of_rows_with_ruled_out_and_infinite_logits(dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(8, vocab, generator=g) * 2
    logits[0] = -math.inf
    logits[1] = -math.inf
    logits[1, vocab // 2] = -3.0                                  # one candidate
    logits[2, ::2] = math.nan
    logits[3] = math.nan
    logits[4, [3, vocab - 1]] = math.inf                          # two that share everything
    logits[5] = torch.finfo(F32).min
    logits[6, :vocab - 7] = -math.inf
    logits[7, torch.randperm(vocab, generator=g)[:vocab - 5]] = -math.inf
    logits = logits.to(dtype).to(DEV)
    scores = (-torch.rand(8, generator=g)).to(DEV)
    for cu in ([0, 1, 2, 3, 4, 5, 6, 7, 8], [0, 4, 8], [0, 8]):
        check_select(logits, scores, cu, 12, run_select(logits, scores, cu, 12))


@pytest.mark.parametrize("count", [1, 4, 12, 33, 64])
@pytest.mark.parametrize("vocab", [64, 3000, 40000])
def test_equal_scores_go_by_beam_and_token(count, vocab):
    """Rows of few values, whole rows that are equal, -0 beside 0: the order is exact."""
    g = torch.Generator().manual_seed(count)
    one = torch.randint(-2, 3, (vocab,), generator=g).float()
    one[one == 0] = torch.where(torch.rand(int((one == 0).sum()), generator=g) < 0.5, 0.0, -0.0)
    rows = [one, one, torch.zeros(vocab), torch.zeros(vocab), one, -one.abs()]
    logits = torch.stack(rows).to(DEV)
    scores = torch.tensor([-1.0, -1.0, -1.0, -1.0, -1.0, -2.0], device=DEV)
    cu = [0, 2, 4, 5, 6]
    got = run_select(logits, scores, cu, count)
    want = plain.select(logits, scores, cu, count)
    for r, expected in enumerate(want):
        assert got[1][r].tolist()[:len(expected)] == [b for _, b, _ in expected]
        assert got[2][r].tolist()[:len(expected)] == [t for _, _, t in expected]


@pytest.mark.parametrize("vocab", [513, 30011])
def test_selection_where_the_best_lie_side_by_side(vocab):
    """Sorted rows: the best are neighbours, a lane's whole chunks."""
    up = torch.linspace(-4, 4, vocab)
    logits = torch.stack([up, up.flip(0), up.roll(vocab // 3)]).to(DEV)
    scores = torch.tensor([0.0, -0.37, -1.1], device=DEV)
    for count in (7, 32, 64):
        check_select(logits, scores, [0, 3], count, run_select(logits, scores, [0, 3], count))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5, 8])
def test_selection_of_rows_that_begin_anywhere(dtype, offset):
    g = torch.Generator().manual_seed(offset)
    wide = torch.full((5, 5021), 99.0, dtype=dtype)
    wide[:, offset:offset + 5003] = (torch.randn(5, 5003, generator=g) * 3).to(dtype)
    logits = wide.to(DEV)[:, offset:offset + 5003]
    scores = (-torch.rand(5, generator=g)).to(DEV)
    check_select(logits, scores, [0, 2, 5], 6, run_select(logits, scores, [0, 2, 5], 6))


def test_selection_of_rows_behind_two_to_the_32():
    """Offsets that pass 32 bits."""
    held = torch.empty(2 * (2**31 + 8) + 3000, dtype=BF16, device=DEV)
    logits = held.as_strided((3, 3000), (2**31 + 8, 1))
    logits.copy_(torch.randn(3, 3000, generator=torch.Generator().manual_seed(1)) * 3)
    scores = torch.tensor([-1.0, -0.5, -0.7], device=DEV)
    check_select(logits, scores, [0, 3], 6, run_select(logits, scores, [0, 3], 6))


def test_selection_tells_scores_of_beams_apart_that_32_bits_do_not():
    """Two beams whose best candidates differ by 2^-30 near 40: the order is the 64-bit one."""
    vocab = 4096
    logits = torch.zeros(2, vocab)
    logits[:, 9] = 20.0
    logits[1, 10:] = -2.0 ** -6                   # a slightly smaller sum, so a slightly better token 9
    total = plain.candidate_scores(logits, torch.tensor([-40.0, -40.0]))
    assert 0 < float(total[1, 9] - total[0, 9]) < 2.0 ** -20
    logits = logits.to(DEV)
    got = run_select(logits, torch.tensor([-40.0, -40.0], device=DEV), [0, 2], 2)
    assert got[1].tolist() == [[1, 0]] and got[2].tolist() == [[9, 9]]


# ------------------------------------------------------------------------------------- reordering
LAYOUTS = [[(F32, 128)], [(BF16, 4096), (BF16, 4096), (F32, 33)], [(BF16, 7), (F32, 1), (torch.int32, 5000), (BF16, 2054)],
           [(F32, 66000)]]


@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
@pytest.mark.parametrize("requests,beams", [(1, 1), (1, 2), (3, 4), (2, 5), (4, 8), (2, 13), (3, 16), (2, 32)])
def test_rows_follow_their_beams(layout, requests, beams):
    """Any parents: several descendants, swaps, rings; entries that name nothing."""
    rng = random.Random(layout * 100 + requests * 10 + beams)
    rows = requests * beams + 3
    held = [torch.randint(-30000, 30000, (rows, n)).to(dtype).to(DEV) for dtype, n in LAYOUTS[layout]]
    order = rng.sample(range(rows), requests * beams)
    slots = [order[r * beams:(r + 1) * beams] for r in range(requests)]
    parents = [[rng.randrange(beams) for _ in range(beams)] for _ in range(requests)]
    parents[0] = [(b + 1) % beams for b in range(beams)]              # a ring
    if requests > 1 and beams > 2:
        parents[1][0], parents[1][1] = -1, beams                      # nothing moves
        slots[1][2] = rows + 5
    want = [plain.reorder(t.cpu(), slots, parents) for t in held]
    set_of = ops().CacheRows(held)
    ops().beam_reorder(set_of, torch.tensor(slots, dtype=torch.int32, device=DEV),
                       torch.tensor(parents, dtype=torch.int32, device=DEV))
    for t, w in zip(held, want):
        assert torch.equal(t.cpu(), w)


@pytest.mark.parametrize("spare,shift", [(0, 0), (1, 0), (2, 2), (4, 4), (12, 1)])
def test_rows_inside_wider_ones_move_alone(spare, shift):
    """Columns of wider slots: what lies beside them stays."""
    wide = torch.randn(11, 700 + spare + shift, device=DEV)
    before = wide.clone()
    parts = [wide[:, shift:shift + 300], wide[:, shift + 300:shift + 700]]
    slots, parents = [[4, 0, 9], [2, 3, 10]], [[2, 0, 1], [0, 0, 1]]
    want = [plain.reorder(p.cpu(), slots, parents) for p in parts]
    ops().beam_reorder(ops().CacheRows(parts), torch.tensor(slots, dtype=torch.int32, device=DEV),
                       torch.tensor(parents, dtype=torch.int32, device=DEV))
    for p, w in zip(parts, want):
        assert torch.equal(p.cpu(), w)
    assert torch.equal(wide[:, :shift], before[:, :shift]) and torch.equal(wide[:, shift + 700:], before[:, shift + 700:])


def test_rows_behind_two_to_the_32():
    """Offsets that pass 32 bits."""
    held = torch.zeros(5, 2**29 + 64, dtype=torch.uint8, device=DEV).view(BF16)       # rows of half a gigabyte and a bit
    held[0, -9:], held[4, -9:] = 3.0, 5.0
    ops().beam_reorder(ops().CacheRows([held]), torch.tensor([[0, 4]], dtype=torch.int32, device=DEV),
                       torch.tensor([[1, 0]], dtype=torch.int32, device=DEV))
    assert held[0, -9:].eq(5.0).all() and held[4, -9:].eq(3.0).all() and held[0, 0] == 0 and held[3, -1] == 0


# ------------------------------------------------------------------------------------- attention
def paged(groups, kv, d, page, dtype, seed, spare=3, poison=True):
    """``groups``: (shared keys, lengths).  Pages in a random order; what no key lies on holds NaN."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    ctx = [n for _, lens in groups for n in lens]
    need = sum(m // page for m, _ in groups) + sum(max(0, -(-n // page) - m // page) for m, lens in groups for n in lens) + spare
    free = list(range(need))
    rng.shuffle(free)
    width = max(1, max(-(-n // page) for n in ctx)) + 1
    k = torch.full((need, kv, page, d), math.nan if poison else 0.0)
    v = torch.full((need, kv, d, page), math.nan if poison else 0.0)
    tables, cu, shared = [], [0], []
    for m, lens in groups:
        common = [free.pop() for _ in range(m // page)]
        for n in lens:
            mine = [free.pop() for _ in range(-(-n // page) - len(common))] if n > 0 else []
            row = (common if n > 0 else []) + mine
            tables.append(row + [-1] * (width - len(row)))
            for j in range(n):
                b = row[j // page]
                if j >= len(common) * page or torch.isnan(k[b, 0, j % page, 0]) or not poison:
                    k[b, :, j % page] = torch.randn(kv, d, generator=g)
                    v[b, :, :, j % page] = torch.randn(kv, d, generator=g)
        cu.append(cu[-1] + len(lens))
        shared.append(m // page * page)
    return k.to(dtype), v.to(dtype), tables, cu, shared, ctx


def run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, scale, sinks=None, cuts=None, widest=None):
    o = ops()
    n = len(ctx)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    q, k, v = q.to(DEV) if not q.is_cuda else q, k.to(DEV), v.to(DEV)
    widest = widest or max(1, max(b - a for a, b in zip(cu, cu[1:])))
    if cuts is None:
        own = max([c - s for s, lo, hi in zip(shared, cu, cu[1:]) for c in ctx[lo:hi]] + [1])
        cuts = o.attn_beams_cuts(q, k, H, KV, d, len(shared), n, widest, max(shared + [0]), own)
    work = o.attn_beams_workspace(n, H, d, cuts, DEV)
    for w in work:
        w.fill_(math.nan)
    out = torch.full((n, H * d), 7.0, dtype=k.dtype, device=DEV)
    o.attn_beams(q, k, v, ints(tables), ints(cu), ints(shared), ints(ctx), out, H, KV, d, scale, widest, cuts, work,
                 sinks=None if sinks is None else sinks.to(DEV))
    return out


def check_attend(out, q, k, v, tables, ctx, H, KV, d, scale, sinks=None):
    """32 bits: a score is a sum of d products, off by about 2^-24 sqrt(d) of its size (up to 8 here, times log2(e)), a
    probability by as much relatively, the output by twice the sum of |p v|: 2^-24 * 16 * 12 * 2 < 2.5e-5 of it.  bf16
    adds the rounding of probabilities (2^-8 of the sum of |p v|) and of the stored output (2^-8 of it)."""
    want, weight = plain.attend(q, k, v, tables, ctx, H, KV, d, scale, sinks)
    bound = 2.5e-5 * weight + 1e-7
    if out.dtype == BF16:
        bound = bound + 2.0 ** -8 * weight + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    for i, n in enumerate(ctx):
        if n == 0:
            assert out[i].eq(0).all()


GROUPS = {
    "one": [(0, [1])],
    "short": [(16, [17, 20, 16, 25])],
    "uneven": [(64, [65, 100, 70]), (0, [5, 1]), (160, [161] * 5), (32, [33])],
    "empty": [(48, [60, 0, 50]), (0, [0, 0]), (16, [0, 30])],
    "exact": [(128, [128, 128, 256]), (256, [256])],
    "long": [(1200, [1300, 1215, 1201, 1500]), (0, [900, 3])],
    "wide": [(96, [100 + i for i in range(17)])],
}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("groups", sorted(GROUPS))
@pytest.mark.parametrize("H,KV,d", [(4, 2, 16), (6, 2, 80), (8, 2, 64), (3, 3, 128), (8, 1, 256), (5, 1, 192), (40, 2, 32)])
def test_attention_behind_shared_pages(dtype, groups, H, KV, d):
    k, v, tables, cu, shared, ctx = paged(GROUPS[groups], KV, d, 16, dtype, 5)
    q = (torch.randn(len(ctx), H * d, generator=torch.Generator().manual_seed(1)) * 1.3).to(dtype)
    sinks = torch.randn(H, generator=torch.Generator().manual_seed(2)) if H == 8 else None
    out = run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, d ** -0.5, sinks)
    check_attend(out, q, k, v, tables, ctx, H, KV, d, d ** -0.5, sinks)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [1, 3, 8, 12, 24, 32])
@pytest.mark.parametrize("cuts", [(1, 1), (3, 2), (64, 64)])
def test_attention_over_pages_of_any_size_in_any_cuts(dtype, page, cuts):
    groups = [(96, [97, 130, 110]), (48, [48, 49]), (0, [200])]
    k, v, tables, cu, shared, ctx = paged(groups, 2, 48, page, dtype, page)
    q = torch.randn(len(ctx), 6 * 48, generator=torch.Generator().manual_seed(page)).to(dtype)
    out = run_attend(q, k, v, tables, cu, shared, ctx, 6, 2, 48, 0.2, cuts=cuts)
    check_attend(out, q, k, v, tables, ctx, 6, 2, 48, 0.2)


@pytest.mark.parametrize("shared", [0, 16, 32, 48])
def test_keys_behind_the_end_of_the_table_are_not_there(shared):
    """Also where the group is said to share them: every key counts once, as the sinks in the denominators show."""
    H, KV, d = 4, 2, 32
    k, v, tables, cu, _, ctx = paged([(32, [40, 33, 32])], KV, d, 16, F32, 3)
    q = torch.randn(len(ctx), H * d, generator=torch.Generator().manual_seed(6))
    sinks = torch.tensor([0.5, 2.0, -1.0, 1.0])
    short = [row[:2] for row in tables]
    out = run_attend(q, k, v, short, cu, [shared], ctx, H, KV, d, 0.3, sinks)
    check_attend(out, q, k, v, short, [32] * 3, H, KV, d, 0.3, sinks)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_lengths_inside_a_page_and_beyond_a_sequence(dtype):
    """Any number of first keys may be shared, the table rows of a group agreeing on them; a sequence that is shorter is read
    by itself, and what others hold behind its end does not reach it."""
    H, KV, d = 4, 2, 32
    k, v, tables, cu, shared, ctx = paged([(64, [70, 90, 66]), (32, [40, 33])], KV, d, 16, dtype, 9)
    q = torch.randn(len(ctx), H * d, generator=torch.Generator().manual_seed(4)).to(dtype)
    for lens in ([61, 5], [0, 31], [64, 32], [1, 17]):
        out = run_attend(q, k, v, tables, cu, lens, ctx, H, KV, d, 0.3)
        check_attend(out, q, k, v, tables, ctx, H, KV, d, 0.3)
    same = [tables[0]] * 3 + tables[3:]
    few = [70, 20, 66] + ctx[3:]
    out = run_attend(q, k, v, same, cu, [64, 32], few, H, KV, d, 0.3)
    check_attend(out, q, k, v, same, few, H, KV, d, 0.3)
    # the first of them the short one, with no more pages than it needs; nobody as long as what is said to be shared
    short = [tables[0][:2] + [-1] * (len(tables[0]) - 2)] + [tables[0]] * 2 + tables[3:]
    for few in ([20, 70, 66] + ctx[3:], [17, 30, 50] + ctx[3:], [0, 0, 40] + ctx[3:]):
        out = run_attend(q, k, v, short, cu, [64, 32], few, H, KV, d, 0.3)
        check_attend(out, q, k, v, short, few, H, KV, d, 0.3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinities_behind_a_short_sequence_stay_with_the_long_ones(dtype):
    H, KV, d = 4, 2, 32
    k, v, tables, cu, shared, ctx = paged([(64, [70, 90, 66])], KV, d, 16, dtype, 9)
    q = torch.randn(3, H * d, generator=torch.Generator().manual_seed(4)).to(dtype)
    v[tables[0][3], :, :, 5], k[tables[0][2], :, 3] = math.inf, math.nan
    few, same = [70, 20, 40], [tables[0]] * 3
    out = run_attend(q, k, v, same, cu, [64], few, H, KV, d, 0.3).cpu()
    assert out[0].isnan().all()
    k[tables[0][2], :, 3] = 0.0
    want, weight = plain.attend(q, k, v, same, few, H, KV, d, 0.3)
    for i in (1, 2):
        bound = 2.5e-5 * weight[i] + 1e-7 + (2.0 ** -8 * (weight[i] + 1.01 * want[i].abs()) if dtype == BF16 else 0.0)
        assert i == 2 or bool(((out[i].double() - want[i]).abs() <= bound).all())
    out = run_attend(q, k, v, same, cu, [64], few, H, KV, d, 0.3).cpu()
    assert not out[0].isfinite().any() and bool(((out[1:].double() - want[1:]).abs() <= 2.5e-5 * weight[1:] + 1e-7 + (
        2.0 ** -8 * (weight[1:] + 1.01 * want[1:].abs()) if dtype == BF16 else 0.0)).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pages_that_are_not_there_and_sequences_outside_groups(dtype):
    H, KV, d = 4, 2, 64
    k, v, tables, cu, shared, ctx = paged([(64, [80, 90]), (0, [100]), (32, [60, 50])], KV, d, 16, dtype, 11)
    tables[0][2] = tables[1][2] = -1
    tables[2][0] = 10**6
    tables[3][3] = -7
    q = torch.randn(len(ctx), H * d, generator=torch.Generator().manual_seed(4)).to(dtype)
    out = run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, 0.3)
    check_attend(out, q, k, v, tables, ctx, H, KV, d, 0.3)
    # the second group unnamed, the third named; lengths past the table; more sequences than the widest group was said to have
    out = run_attend(q, k, v, tables, [0, 2], [64], ctx, H, KV, d, 0.3, widest=1)
    check_attend(out, q, k, v, tables, ctx, H, KV, d, 0.3)
    far = [c + 10**6 for c in ctx]
    out = run_attend(q, k.nan_to_num(1.0), v.nan_to_num(2.0), tables, cu, shared, far, H, KV, d, 0.3, cuts=(2, 2))
    check_attend(out, q, k.nan_to_num(1.0), v.nan_to_num(2.0), tables, far, H, KV, d, 0.3)


@pytest.mark.parametrize("page", [16, 12])
def test_pages_behind_two_to_the_32(page):
    """Offsets that pass 32 bits: the pages of a small cache at the end of a large one."""
    H, KV, d = 8, 2, 64
    k, v, tables, cu, shared, ctx = paged([(48, [60, 100, 49]), (0, [30])], KV, d, page, BF16, 8)
    first = 2**32 // (KV * page * d) + 5
    far = [torch.empty(first + t.shape[0], *t.shape[1:], dtype=BF16, device=DEV) for t in (k, v)]
    for held, t in zip(far, (k, v)):
        held[0] = math.nan
        held[first:].copy_(t)
    q = torch.randn(len(ctx), H * d, generator=torch.Generator().manual_seed(4)).to(BF16)
    moved = [[first + p if p >= 0 else p for p in row] for row in tables]
    out = run_attend(q, *far, moved, cu, shared, ctx, H, KV, d, 0.2)
    check_attend(out, q, k, v, tables, ctx, H, KV, d, 0.2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_scores_and_rows_of_wider_tensors(dtype):
    """Scores far apart (one key takes all), and q as columns of a wider projection."""
    H, KV, d = 8, 2, 64
    k, v, tables, cu, shared, ctx = paged([(320, [330, 400, 321])], KV, d, 16, dtype, 3)
    wide = (torch.randn(3, H * d + 2 * KV * d, generator=torch.Generator().manual_seed(8))).to(dtype).to(DEV)
    q = wide[:, :H * d]
    for scale in (0.0, 0.125, 8.0):
        out = run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, scale)
        want, weight = plain.attend(q, k, v, tables, ctx, H, KV, d, scale)
        # a score of size 250 * scale is off by 2^-20 of it: so are, relatively, the probabilities
        bound = (2.5e-5 + 2.0 ** -19 * 250 * scale) * weight + 1e-7
        if dtype == BF16:
            bound = bound + 2.0 ** -8 * weight + 2.0 ** -8 * want.abs() * 1.01
        assert bool(((out.cpu().double() - want).abs() <= bound).all())


def test_not_a_number_stays_in_its_row():
    H, KV, d = 4, 2, 64
    k, v, tables, cu, shared, ctx = paged([(64, [80, 90, 70])], KV, d, 16, F32, 3)
    q = torch.randn(3, H * d, generator=torch.Generator().manual_seed(8))
    q[1, d:2 * d] = math.nan
    out = run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, 0.1).cpu()
    assert out[1, d:2 * d].isnan().all() and int(out.isnan().sum()) == d
    want, _ = plain.attend(q, k, v, tables, ctx, H, KV, d, 0.1)
    assert torch.allclose(out[0].double(), want[0], atol=1e-5)


def test_attention_agrees_with_the_decode_kernel():
    """The same pages through ``attn_decode``, which reads every sequence's keys by themselves."""
    H, KV, d = 32, 8, 64
    k, v, tables, cu, shared, ctx = paged([(512, [600, 530, 700, 513]), (16, [40, 20])], KV, d, 16, BF16, 21)
    q = torch.randn(len(ctx), H * d, generator=torch.Generator().manual_seed(8)).to(BF16)
    out = run_attend(q, k, v, tables, cu, shared, ctx, H, KV, d, 0.125)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    other = torch.empty_like(out)
    n = len(ctx)
    ops().attn_decode(q.to(DEV), k.to(DEV), v.to(DEV), ints(tables), None, n, ints(list(range(n + 1))), ints(ctx), other, H, KV, d,
                      0.125, token_is_seq=True)
    check_attend(out, q, k, v, tables, ctx, H, KV, d, 0.125)
    check_attend(other, q, k, v, tables, ctx, H, KV, d, 0.125)


# ------------------------------------------------------------------------------------- together
def one_step(state):
    """Attention of the beams, selection from the logits a (fixed) head makes of it, and the beams' rows following."""
    o = ops()
    o.attn_beams(state["q"], state["k"], state["v"], state["table"], state["cu"], state["shared"], state["ctx"], state["out"],
                 state["H"], state["KV"], state["d"], 0.2, 4, state["cuts"], state["work"])
    torch.mm(state["out"], state["head"], out=state["logits"])
    o.beam_select(state["logits"], state["scores"], state["cu"], *state["picked"], state["select_work"])
    state["parents"].copy_(state["picked"][1][:, :4])
    o.beam_reorder(state["rows"], state["slots"], state["parents"])


def together(seed):
    H, KV, d, page, vocab = 8, 2, 64, 16, 5000
    groups = [(160, [161, 170, 165, 175]), (64, [65, 66, 70, 79])]
    k, v, tables, cu, shared, ctx = paged(groups, KV, d, page, F32, seed, poison=False)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(seed)
    s = {"H": H, "KV": KV, "d": d, "k": k.to(DEV), "v": v.to(DEV), "table": ints(tables), "cu": ints(cu), "shared": ints(shared),
         "ctx": ints(ctx), "q": torch.randn(8, H * d, generator=g).to(DEV), "head": torch.randn(H * d, vocab, generator=g).to(DEV),
         "scores": (-torch.rand(8, generator=g)).to(DEV), "out": torch.zeros(8, H * d, device=DEV),
         "logits": torch.zeros(8, vocab, device=DEV), "parents": torch.zeros(2, 4, dtype=torch.int32, device=DEV),
         "slots": ints([[t[c // page] for t, c in zip(tables[i:i + 4], ctx[i:i + 4])] for i in (0, 4)])}
    s["rows"] = ops().CacheRows([s["k"], s["v"]])
    s["cuts"] = ops().attn_beams_cuts(s["q"], s["k"], H, KV, d, 2, 8, 4, 160, 15)
    s["work"] = ops().attn_beams_workspace(8, H, d, s["cuts"], DEV)
    s["picked"] = (torch.zeros(2, 8, device=DEV), torch.zeros(2, 8, dtype=torch.int32, device=DEV), torch.zeros(2, 8, dtype=torch.int32, device=DEV))
    s["select_work"] = ops().beam_select_workspace(8, vocab, 8, DEV)
    return s, (tables, cu, ctx)


def test_a_run_of_all_three_steps_against_the_plain_one():
    s, (tables, cu, ctx) = together(31)
    for _ in range(3):
        k0, v0 = s["k"].cpu(), s["v"].cpu()
        one_step(s)
        check_attend(s["out"], s["q"], k0, v0, tables, ctx, s["H"], s["KV"], s["d"], 0.2)
        check_select(s["logits"], s["scores"], cu, 8, s["picked"])
        slots, parents = s["slots"].tolist(), s["picked"][1][:, :4].tolist()
        assert torch.equal(s["k"].cpu(), plain.reorder(k0, slots, parents))
        assert torch.equal(s["v"].cpu(), plain.reorder(v0, slots, parents))


def test_captured_steps_give_what_eager_ones_give():
    """Replayed several times with eager work between, with other inputs in the same memory; two graphs with workspaces of
    their own; another stream than the default one."""
    a, b = together(1)[0], together(2)[0]
    graphs = []
    for s in (a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one_step(s)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one_step(s)
        graphs.append(graph)
    for turn in range(4):
        for s, graph in zip((a, b), graphs):
            twin = together(1)[0]
            s["q"].normal_()
            for name in ("q", "k", "v", "scores", "head", "table", "ctx", "cu", "shared", "slots"):
                twin[name].copy_(s[name])
            one_step(twin)
            graph.replay()
            torch.cuda.synchronize()
            for name in ("out", "logits", "k", "v"):
                assert torch.equal(s[name], twin[name]), (turn, name)
            assert all(torch.equal(x, y) for x, y in zip(s["picked"], twin["picked"]))


def test_operands_of_another_kind_are_refused():
    o = ops()
    logits, scores = torch.zeros(2, 50, device=DEV), torch.zeros(2, device=DEV)
    with pytest.raises(o.KernelError):
        run_select(logits.half(), scores, [0, 2], 2)
    with pytest.raises(o.KernelError):
        run_select(logits.cpu(), scores, [0, 2], 2)
    with pytest.raises(o.KernelError):
        run_select(logits, scores, [0, 2], 4, work=o.beam_select_workspace(1, 50, 4, DEV))
