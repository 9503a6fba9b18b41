"""Beam search without a GPU: what the operators refuse, pages that beams share and branch off, the host's choice of beams
against the definition, and batches whose sequences share pages."""

from __future__ import annotations

import math
import random

import pytest
import torch

from kvforge_amd.cache import RELEASED, CacheGroup, CacheManager, NoFreeBlocksError
from kvforge_amd.cache.manager import common_start
from kvforge_amd.engine.batch import DecodeShape, MetaBuffers, SharedShape, Step, StepEntry, fill_step
from kvforge_amd.engine.beams import BeamSearcher, Search
from kvforge_amd.kernels import ops
from kvforge_amd.parts import attention_pages
from kvforge_amd.parts.attention import SHARED_FROM, PagedAttention
from kvforge_amd.sampling.params import BeamParams
from tests.plain import beams as plain

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32


# ------------------------------------------------------------------------------------- refusals
@pytest.fixture
def launched(monkeypatch):
    """Tensors of the CPU pass for the GPU's, and a launch only says that it was made."""
    made = []
    monkeypatch.setattr(ops, "_check", ops._check_in_python)
    monkeypatch.setattr(ops, "_placed", ops._placed_in_python)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(ops, "compute_units", lambda device: 256)

    def fn(module, name, argtypes):
        def call(*args):
            made.append(name)
            return 4096 if name == "kvf_beam_tile_bytes" else 1 + (args[3] > 16) if name == "kvf_attn_beams_row_tiles" else 0
        return call
    monkeypatch.setattr(ops, "_fn", fn)
    ops._attn_beams_tiles.cache_clear()
    yield made
    ops._attn_beams_tiles.cache_clear()


def select_args(rows=6, vocab=40, requests=2, count=4, dtype=F32):
    return dict(logits=torch.zeros(rows, vocab, dtype=dtype), scores=torch.zeros(rows), cu_beams=torch.tensor([0, 3, 6], dtype=I32)[:requests + 1],
                out_scores=torch.zeros(requests, count), out_beams=torch.zeros(requests, count, dtype=I32),
                out_tokens=torch.zeros(requests, count, dtype=I32), workspace=ops.beam_select_workspace(rows, vocab, count, "cpu"))


def test_selection_refuses_what_its_kernels_do_not_take(launched):
    ops.beam_select(**select_args())
    ops.beam_select(**select_args(dtype=BF16))
    assert launched == ["kvf_beam_select"] * 2
    good = select_args()
    wide = torch.zeros(6, 80)
    bad = [dict(logits=good["logits"].half()), dict(logits=good["logits"][0]), dict(logits=wide[:, ::2]), dict(logits=torch.zeros(6, 0)),
           dict(logits=torch.zeros(40).expand(6, 40)), dict(scores=torch.zeros(5)), dict(scores=good["scores"].double()),
           dict(cu_beams=good["cu_beams"].long()), dict(cu_beams=good["cu_beams"][:0]), dict(cu_beams=good["cu_beams"][:2]),
           dict(out_beams=torch.zeros(2, 5, dtype=I32)), dict(out_tokens=torch.zeros(2, 4)), dict(out_scores=torch.zeros(2, 4).bfloat16()),
           dict(out_scores=torch.zeros(2, 0), out_beams=torch.zeros(2, 0, dtype=I32), out_tokens=torch.zeros(2, 0, dtype=I32)),
           {k: v for k, v in select_args(count=65).items() if k.startswith("out")}, dict(workspace=ops.beam_select_workspace(1, 40, 4, "cpu")),
           dict(out_tokens=good["out_beams"]), dict(out_scores=good["workspace"][1][:8].view(2, 4)),
           dict(out_beams=good["cu_beams"][:0].new_zeros(8).view(2, 4).t().contiguous())]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.beam_select(**{**good, **change})
    with pytest.raises(ops.KernelError):
        ops.beam_select(**{**good, "logits": torch.zeros(1, 40).expand(70000, 40)})
    with pytest.raises(ops.KernelError, match="more than the kernel counts"):
        big = select_args(rows=1, vocab=40, requests=1, count=64)
        ops.beam_select(**{**big, "logits": torch.zeros(1, 4096 * 1025, dtype=BF16), "cu_beams": torch.tensor([0, 1], dtype=I32)})
    assert len(launched) == 2


def test_reordering_refuses_what_its_kernels_do_not_take(launched):
    held = [torch.zeros(9, 4, 5), torch.zeros(9, 33, dtype=BF16)]
    rows = ops.CacheRows(held)
    assert rows.tiles.shape == (2, 3) and rows.rows == 9
    slots = torch.zeros(2, 4, dtype=I32)
    ops.beam_reorder(rows, slots, slots.clone())
    assert launched.count("kvf_beam_reorder") == 1
    for s, p in ((slots.long(), slots), (slots, slots[:, :3]), (slots[0], slots[0]), (torch.zeros(2, 33, dtype=I32),) * 2,
                 (torch.zeros(70000, 1, dtype=I32),) * 2, (torch.zeros(2, 0, dtype=I32),) * 2):
        with pytest.raises(ops.KernelError):
            ops.beam_reorder(rows, s, p)
    wide = torch.zeros(9, 50)
    for tensors in ([], [torch.zeros(9)], [torch.zeros(9, 4), torch.zeros(8, 4)], [torch.zeros(9, 8)[:, ::2]], [torch.zeros(9, 4, dtype=torch.uint8)],
                    [torch.zeros(4).expand(9, 4)], [wide, wide], [wide[:, :20], wide[:, 19:]], [wide[:, :20], wide[:8, 20:]], [torch.zeros(0, 4)],
                    [wide[:, :20], wide.view(18, 25)[:9, :]]):
        with pytest.raises(ops.KernelError):
            ops.CacheRows(tensors)
    assert ops.CacheRows([wide[:, :20], wide[:, 20:]]).tiles[:, 2].tolist() == [80 + (4 << 32) if (wide.data_ptr() % 8 or 200 % 8) else 80 + (8 << 32),
                                                                                120 + (8 << 32)]


def attend_args(n=4, H=4, KV=2, d=32, page=16, dtype=F32):
    return dict(q=torch.zeros(n, H * d, dtype=dtype), k_pages=torch.zeros(7, KV, page, d, dtype=dtype),
                v_pages=torch.zeros(7, KV, d, page, dtype=dtype), block_table=torch.zeros(n, 3, dtype=I32),
                cu_groups=torch.tensor([0, 3, 4], dtype=I32), shared_lens=torch.zeros(2, dtype=I32), ctx_lens=torch.zeros(n, dtype=I32),
                out=torch.zeros(n, H * d, dtype=dtype), num_heads=H, num_kv_heads=KV, head_dim=d, scale=0.1, widest=3, cuts=(2, 1),
                workspace=ops.attn_beams_workspace(n, H, d, (2, 1), "cpu"))


def test_attention_refuses_what_its_kernels_do_not_take(launched):
    ops.attn_beams(**attend_args())
    ops.attn_beams(**attend_args(dtype=BF16), sinks=torch.zeros(4))
    assert launched.count("kvf_attn_beams") == 2
    good = attend_args()
    bad = [dict(num_kv_heads=3), dict(num_kv_heads=0), dict(head_dim=24), dict(head_dim=272), dict(q=good["q"].half()),
           dict(q=torch.zeros(4, 127)), dict(q=torch.zeros(4, 130)[:, :128]), dict(q=torch.zeros(4, 256)[:, ::2]), dict(q=torch.zeros(129 * 4)[1:].view(-1)[:512].view(4, 128)),
           dict(k_pages=good["k_pages"].bfloat16()), dict(v_pages=good["k_pages"]), dict(block_table=torch.zeros(3, 3, dtype=I32)),
           dict(cu_groups=good["cu_groups"][:0]), dict(shared_lens=torch.zeros(3, dtype=I32)), dict(ctx_lens=torch.zeros(4)),
           dict(out=torch.zeros(5, 128)), dict(out=good["q"]), dict(widest=0), dict(cuts=(65, 1)), dict(cuts=(2, 0)), dict(cuts=(-1, 1)),
           dict(cuts=(3, 1)), dict(sinks=torch.zeros(3)), dict(sinks=torch.zeros(4).bfloat16()),
           dict(workspace=(good["workspace"][0], good["workspace"][0][:24])),
           dict(block_table=torch.zeros(1, 1, dtype=I32).expand(4, 2**28).as_strided((4, 2**28), (0, 0)))]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.attn_beams(**{**good, **change})
    assert launched.count("kvf_attn_beams") == 2


def test_attention_refuses_more_sequences_and_wider_strides_than_it_counts(launched):
    ops.attn_beams(**attend_args(n=2, dtype=BF16))
    apart = torch.empty(2**31 + 128, dtype=BF16).as_strided((2, 128), (2**31, 1))        # (nothing of it is touched)
    many = torch.empty(2**21, 4 * 16, dtype=BF16)
    for change in (dict(q=apart), dict(q=many, head_dim=16)):
        with pytest.raises(ops.KernelError, match="more than the kernel counts"):
            ops.attn_beams(**{**attend_args(n=2, dtype=BF16), **change})
    assert launched.count("kvf_attn_beams") == 1


def test_cuts_fit_the_chip_and_the_keys(launched):
    q, k = torch.zeros(1, 4, dtype=BF16), torch.zeros(1, 8, 16, 64, dtype=BF16)
    cuts = lambda *a: ops.attn_beams_cuts(q, k, 32, 8, 64, *a)
    assert cuts(1, 4, 4, 300, 20) == (3, 1)                 # a round of the waves each
    assert cuts(0, 4, 1, 0, 1000) == (0, 16) and cuts(2, 4, 4, 0, 1) == (0, 1)
    assert cuts(4, 16, 4, 100000, 20) == (6, 1) and cuts(16, 64, 4, 100000, 20) == (2, 1)       # 32 and 128 items of one tile
    assert cuts(4, 32, 8, 100000, 20) == (8, 1) and cuts(16, 128, 8, 100000, 20) == (2, 1)      # and of two
    assert cuts(100, 400, 4, 100000, 300) == (1, 1)
    assert all(1 <= c <= 64 for n in (1, 7, 300) for c in cuts(n, 4 * n, 4, 10**6, 10**6))


def test_placement_is_asked_of_the_current_device(launched, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call, args in ((ops.beam_select, select_args()), (ops.attn_beams, attend_args())):
        with pytest.raises(ops.KernelError, match="current device is 1"):
            call(**args)


# ------------------------------------------------------------------------------------- pages
FULL, WINDOW = CacheGroup((0,), attention_pages(1, 16)), CacheGroup((1,), attention_pages(1, 16), window=6)


def manager(blocks=40, slots=0):
    return CacheManager(4, [FULL, WINDOW], blocks, num_state_slots=slots)


def held(m):
    """Pages by how many tables name them, per group: what the pools have to count."""
    out = []
    for g, pool in enumerate(m.pools):
        named: dict[int, int] = {}
        for table in m._tables[g].values():
            for b in table:
                if b != RELEASED:
                    named[b] = named.get(b, 0) + 1
        assert all(pool.ref_count(b) == named.get(b, 0) for b in range(pool.num_blocks))
        assert pool.num_used == len(named)
        out.append(named)
    return out


def test_a_branch_shares_what_is_filled_and_owns_what_is_not():
    m = manager(slots=4)
    m.allocate("a", 10)
    serial = m.serial("a")
    m.branch("b", "a", 10)
    a, b = m.block_table("a"), m.block_table("b")
    assert b[:2] == a[:2] and b[2] != a[2] and len(b) == 3 and m.num_tokens("b") == 10
    assert m.slots.slot("b") != m.slots.slot("a") and m.serial("b") != serial and m.serial("a") == serial
    held(m)
    assert m.shared_pages(["a", "b"]) == 2
    m.append_slots("a", 12, 10)
    m.branch("c", "a", 12)                       # nothing is being filled: every page is shared
    assert m.block_table("c") == m.block_table("a") and m.shared_pages(["a", "c"]) == 3
    m.append_slots("c", 13, 12)
    assert m.block_table("c")[:3] == m.block_table("a") and m.shared_pages(["a", "b", "c"]) == 2
    slot = m.slots.slot("b")
    serial = m.serial("b")
    m.free("a")
    held(m)
    m.append_slots("c", 14, 13)
    m.branch("b", "c", 14)                       # a place is taken anew: what it held goes back
    assert m.slots.slot("b") == slot and m.serial("b") != serial and m.block_table("b")[:3] == m.block_table("c")[:3]
    held(m)
    m.free("b")
    m.free("c")
    assert all(p.num_free == p.num_blocks for p in m.pools) and m.slots.num_free == 4


def test_branches_behind_a_window():
    m = manager()
    m.allocate("a", 18)
    m.release_behind("a", 18)
    assert m.block_table("a", 1)[:3] == [RELEASED] * 3
    m.branch("b", "a", 18)
    assert m.block_table("b", 1)[:3] == [RELEASED] * 3 and m.block_table("b", 1)[3] == m.block_table("a", 1)[3]
    held(m)
    for rid in ("a", "b"):
        m.append_slots(rid, 24, 18)
        m.release_behind(rid, 24)
    held(m)
    assert m.shared_pages(["a", "b"]) == 4       # windows are not asked


def test_branches_that_cannot_be_are_refused_whole():
    m = CacheManager(4, [FULL], 4)
    m.allocate("a", 10)
    with pytest.raises(ValueError):
        m.branch("a", "a", 10)
    with pytest.raises(ValueError):
        m.branch("b", "a", 11)
    with pytest.raises(ValueError):
        m.branch("b", "a", 8)                    # the table holds more than that
    m.allocate("x", 1)
    before = held(m), dict(m._num_tokens)
    with pytest.raises(NoFreeBlocksError):
        m.branch("b", "a", 10)
    assert (held(m), dict(m._num_tokens)) == before and not m.has_request("b")
    m.branch("x", "a", 10)                       # the page that it holds serves
    held(m)


@pytest.mark.parametrize("seed", range(6))
def test_no_page_is_lost_in_random_searches(seed):
    rng = random.Random(seed)
    m = manager(200, slots=16)
    live: dict[str, int] = {}
    for turn in range(300):
        if len(live) < 8 and rng.random() < 0.3:
            rid = f"r{turn}"
            live[rid] = rng.randint(1, 20)
            m.allocate(rid, live[rid])
        elif live and rng.random() < 0.2:
            rid = rng.choice(sorted(live))
            m.free(rid)
            del live[rid]
        elif len(live) > 1 and rng.random() < 0.5:
            parent, child = rng.sample(sorted(live), 2)
            m.branch(child, parent, live[parent])
            live[child] = live[parent]
        elif live:
            rid = rng.choice(sorted(live))
            n = rng.randint(1, 3)
            m.append_slots(rid, live[rid] + n, live[rid])
            live[rid] += n
            m.release_behind(rid, live[rid])
        tables = held(m)
        # a page that is being filled has one owner
        for rid, n in live.items():
            if n % 4:
                assert all(named[m.block_table(rid, g)[-1]] == 1 for g, named in enumerate(tables))
    for rid in live:
        m.free(rid)
    assert all(p.num_free == p.num_blocks for p in m.pools) and m.slots.num_free == 16


def test_the_common_start_of_two_lists():
    rng = random.Random(1)
    for _ in range(400):
        a = [rng.randrange(3) for _ in range(rng.randrange(9))]
        b = a[:rng.randrange(len(a) + 1)] + [rng.randrange(3) for _ in range(rng.randrange(4))]
        want = next((i for i, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))
        assert common_start(a, b) == common_start(b, a) == want


# ------------------------------------------------------------------------------------- the choice of beams
def toy(vocab, seed):
    """Logits by the last two tokens."""
    table = torch.randn(vocab, vocab, vocab, generator=torch.Generator().manual_seed(seed)) * 2
    return lambda tokens: table[tokens[-2] if len(tokens) > 1 else 0, tokens[-1]]


@pytest.mark.parametrize("width", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("stops,early,penalty", [((), False, 1.0), ((3,), False, 1.0), ((0, 5), True, 0.0), ((1,), False, 2.0), (tuple(range(12)), False, 0.7)])
def test_the_search_is_the_definition(width, stops, early, penalty):
    """Candidates as the device would give them; every place's history is followed as its pages would be."""
    vocab, prompt = 13, [2, 7]
    for seed in range(4):
        logits = toy(vocab, seed)
        params = BeamParams(width=width, max_tokens=9, length_penalty=penalty, early_stopping=early)
        search = Search(prompt, params, set(stops), 9)
        memory = {0: list(prompt)}
        while not search.done:
            rows = torch.stack([logits(memory[p]) for p in search.places])
            scores = torch.tensor([search.log_probs[p] for p in search.places], dtype=torch.float64)
            found = plain.select(rows, scores, [0, len(search.places)], 2 * width)[0]
            parents = search.advance(found)
            assert sorted(parents) == search.places and all(0 <= p < width for p in search.places)
            # a parent with descendants keeps its place, so nothing that is copied from is written
            assert all(parents[p] == p for p in parents.values()) or search.done
            memory = {to: memory[p] + [search.tokens[to][-1]] for to, p in parents.items()}
            assert all(memory[p] == prompt + search.tokens[p] for p in search.places)
        want, _ = plain.search(logits, prompt, width, 9, penalty, early, set(stops))
        got = search.output().sequences
        assert [(s.output_token_ids, s.finish_reason.value) for s in got] == [(t, r) for t, _, _, r in want]
        assert all(abs(s.log_prob - p) < 1e-9 and abs(s.score - q) < 1e-9 for s, (_, p, q, _) in zip(got, want))


def test_parameters_that_make_no_search_are_refused():
    for bad in (dict(width=0), dict(width=33), dict(max_tokens=0), dict(num_return=0), dict(width=2, num_return=3)):
        with pytest.raises(ValueError):
            BeamParams(**bad)
    few = Search([1], BeamParams(width=3, num_return=2), set(), 1)
    few.advance([(-1.0, 0, 4), (-2.0, 0, 5), (-3.0, 0, 6)])
    assert few.done and [s.output_token_ids for s in few.output().sequences] == [[4], [5]]
    none = Search([1], BeamParams(width=3), set(), 5)
    none.advance([])
    assert none.done and none.output().sequences == []


def test_pages_that_a_search_can_come_to_hold():
    searcher = BeamSearcher.__new__(BeamSearcher)
    searcher.cache = CacheManager(4, [FULL], 10)
    assert searcher.pages_needed(8, BeamParams(width=3), 4) == 2 + 3
    assert searcher.pages_needed(9, BeamParams(width=3), 4) == 2 + 3 * 2
    assert searcher.pages_needed(3, BeamParams(width=1), 1) == 1


# ------------------------------------------------------------------------------------- batches
def filled(shared, starts=(9, 9, 9, 4, 4), pad_to=None):
    tables = {f"r{i}": [10 * i + p for p in range(6)] for i in range(len(starts))}
    meta = MetaBuffers(32, 8, [6], "cpu")
    step = Step()
    entries = [StepEntry(f"r{i}", [1], s, "last") for i, s in enumerate(starts)]
    fill_step(step, meta, entries, lambda r, g: tables[r], lambda r: -1, 4, pad_to, [False], lambda r: 0, shared=shared)
    return step


def test_a_batch_says_which_sequences_share_pages():
    step = filled([(3, 8), (2, 0)])
    assert step.shared.cu_groups.tolist() == [0, 3, 5] and step.shared.shared_lens.tolist() == [8, 0]
    assert step.shared.shape == step.decode_shape.groups == SharedShape(2, 3, 512, 64)
    assert filled(None).shared is None and filled(None).decode_shape.groups is None
    assert filled([(5, 0)]).shared.shape == SharedShape(1, 5, 0, 64)
    for bad in ([(3, 8)], [(3, 11), (2, 0)], [(5, 8)], [(3, -1), (2, 0)], [(0, 0), (5, 0)]):
        with pytest.raises(ValueError):
            filled(bad)
    with pytest.raises(ValueError):
        filled([(5, 0)], pad_to=8)


def test_which_layers_read_shared_pages_once():
    def layer(dtype=BF16, **kw):
        part = PagedAttention("a", 64, 4, 2, 16, None, **kw)
        part.w_qkv = torch.zeros(1, dtype=dtype)
        return part
    far, near = SharedShape(1, 4, SHARED_FROM + 512, 64), SharedShape(1, 4, SHARED_FROM, 64)
    shape = lambda groups: DecodeShape(4, 640, 2400, groups)
    assert layer().launch_key(shape(far)) == far and layer().launch_key(shape(near)) == (1, 1) == layer().launch_key(shape(None))
    assert layer(F32).launch_key(shape(near)) == near
    assert layer(F32).launch_key(shape(SharedShape(1, 4, 0, 64))) == (1, 1)
    assert layer(sink="s").launch_key(shape(far)) == far
    for kw in (dict(window=600), dict(chunk=600), dict(score_slopes=[1.0] * 4), dict(score_cap=5.0), dict(distance_bias=("d", 50.0), distance_buckets=8)):
        assert layer(**kw).launch_key(shape(far)) == (1, 1), kw
