"""Whole beam searches without a GPU, over a toy model that keeps its tokens in the cache's pages and slots and reads them back
from there: what a step reads has to be what its beams have seen, however beams branch, end, and come to be one or many."""

from __future__ import annotations

import random
from types import SimpleNamespace

import pytest
import torch

from kvforge_amd.cache import CacheGroup, CacheManager
from kvforge_amd.engine.beams import BeamSearcher
from kvforge_amd.kernels import ops
from kvforge_amd.parts import attention_pages
from kvforge_amd.sampling.params import BeamParams
from tests.plain import beam_search, beams as plain

VOCAB, NONE = 13, -1


class PagedToy:
    """A runner whose model keeps a token's number in its page and in the request's slot, and whose logits go by the last two tokens
    that it finds there.  Steps with groups read the shared keys from the first sequence's pages."""

    def __init__(self, seed=0, block=4, blocks=120, seqs=16, window=None, tokens=9) -> None:
        groups = [CacheGroup((0,), attention_pages(1, 16))]
        if window:
            groups.append(CacheGroup((1,), attention_pages(1, 16), window=window))
        self.cache, self.device, self.window = CacheManager(block, groups, blocks, num_state_slots=seqs), "cpu", window
        self.pages = [{"k": torch.full((blocks, block), NONE)} for _ in groups]
        self.storage = SimpleNamespace(pages=self.pages)
        self.seen = torch.full((seqs, 64), NONE)
        self.states = SimpleNamespace(tensors={"seen": self.seen})
        self.meta = SimpleNamespace(max_seqs=seqs, max_tokens=tokens)
        self.model = SimpleNamespace(config=SimpleNamespace(vocab_size=VOCAB))
        self.max_model_len = 64
        self.table = torch.randn(VOCAB, VOCAB, VOCAB, generator=torch.Generator().manual_seed(seed)) * 2
        self.widths: list[int] = []         # sequences of every group of every step

    def after(self, tokens):
        return self.table[tokens[-2] if len(tokens) > 1 else 0, tokens[-1]]

    def read(self, table, group, lo, hi):
        bs = self.cache.block_size
        return [int(self.pages[group]["k"][table[j // bs], j % bs]) for j in range(lo, hi)]

    def step(self, entries, shared=None):
        cache, bs, logits = self.cache, self.cache.block_size, []
        assert len(entries) <= self.meta.max_seqs and sum(len(e.token_ids) for e in entries) <= self.meta.max_tokens
        for e in entries:
            for j, t in enumerate(e.token_ids, e.start_pos):
                for g in range(cache.num_groups):
                    table = cache.block_table(e.request_id, g)
                    assert cache.pools[g].ref_count(table[j // bs]) == 1, "a page that others hold is written"
                    self.pages[g]["k"][table[j // bs], j % bs] = t
                self.seen[cache.slots.slot(e.request_id), j] = t
        of = [(first, keys) for first, n, keys in grouped(shared or [(1, 0)] * len(entries)) for _ in range(n)]
        self.widths += [n for n, _ in shared or []]
        for e, (first, keys) in zip(entries, of):
            if e.want != "last":
                continue
            n = e.start_pos + len(e.token_ids)
            assert keys <= e.start_pos
            seen = self.seen[cache.slots.slot(e.request_id), :n].tolist()
            own, held = cache.block_table(e.request_id), cache.block_table(entries[first].request_id)
            assert self.read(held, 0, 0, keys) + self.read(own, 0, keys, n) == seen
            if self.window:
                assert self.read(cache.block_table(e.request_id, 1), 1, max(0, n - self.window), n) == seen[max(0, n - self.window):]
            logits.append(self.after(seen))
        return torch.stack(logits) if logits else torch.empty(0, VOCAB)


def grouped(shared):
    first = 0
    for n, keys in shared:
        yield first, n, keys
        first += n


@pytest.fixture
def on_the_cpu(monkeypatch):
    def reorder(rows, slots, parents):
        for t in rows:
            t.copy_(plain.reorder(t, slots.tolist(), parents.tolist()))
    monkeypatch.setattr(ops, "CacheRows", list)
    monkeypatch.setattr(ops, "beam_reorder", reorder)


def select_by(keep=lambda turn, candidates: candidates):
    """Selection by its definition, of whose candidates (all there are of a request) ``keep`` leaves some."""
    turns = []

    def select(logits, searches, count, ruled_out=None):
        if ruled_out is not None:
            out = set(ruled_out.tolist())
            return [[c for c in found if c[2] not in out][:count] for found in plain.select(logits, *rows_of(searches), VOCAB * 16)]
        turns.append(len(turns))
        return [keep(turns[-1], found)[:count] for found in plain.select(logits, *rows_of(searches), VOCAB * 16)]
    return select


def rows_of(searches):
    cu = [0]
    for s in searches:
        cu.append(cu[-1] + len(s.places))
    return torch.tensor([s.log_probs[p] for s in searches for p in s.places], dtype=torch.float64), cu


def empty(cache):
    assert all(p.num_free == p.num_blocks for p in cache.pools) and cache.slots.num_free == cache.slots.num_slots


@pytest.mark.parametrize("window", [None, 6])
@pytest.mark.parametrize("lives", [(1, 2, 2, 4, 4), (4, 1, 3, 3, 3), (2, 1, 1, 2, 2, 2), (1, 1, 1, 4), (3, 1, 4, 1, 4, 1, 4)])
@pytest.mark.parametrize("length", [3, 4, 5, 6, 7])
def test_beams_that_become_one_and_many_again(on_the_cpu, lives, length, window):
    """``lives``: how many candidates there are, step by step and round and round; prompts end anywhere in a page of four."""
    runner = PagedToy(length, window=window)
    searcher = BeamSearcher(runner)
    rng = random.Random(length)

    def keep(turn, candidates):
        # (any of the best few: parents of one descendant and of several)
        return sorted(rng.sample(candidates[:6], min(lives[turn % len(lives)], len(candidates))), key=candidates.index)
    searcher._select = select_by(keep)
    prompts = [[rng.randrange(VOCAB) for _ in range(n)] for n in (length, length + 9)]
    found = searcher.run(prompts, BeamParams(width=4, max_tokens=17), set())
    assert all(s.done and s.ended for s in found)
    assert {1, max(lives)} <= set(runner.widths)
    empty(runner.cache)


def test_sharing_that_is_known_is_of_filled_pages():
    """A beam alone shares its whole table with itself; behind a branch the page that it was filling is two."""
    m = CacheManager(4, [CacheGroup((0,), attention_pages(1, 16))], 20)
    m.allocate("a", 7)
    assert m.shared_pages(["a"]) == 2
    m.branch("b", "a", 7)
    known = min(2, 7 // 4)
    assert m.shared_pages(["a", "b"], known) == m.shared_pages(["a", "b"]) == 1
    for rid in ("a", "b"):
        m.append_slots(rid, 9, 7)
    assert m.shared_pages(["a", "b"], known) == 1
    m.branch("b", "a", 9)
    assert m.shared_pages(["a", "b"], known) == m.shared_pages(["a", "b"]) == 2


# ------------------------------------------------------------------------------------- several stop tokens
@pytest.mark.parametrize("width,stops", [(1, (3, 8)), (2, (0, 5)), (2, (1, 4, 9)), (4, (0, 3, 6, 9)), (3, tuple(range(12))), (5, tuple(range(11))),
                                         (4, tuple(range(0, 13, 2))), (2, tuple(range(13)))])
@pytest.mark.parametrize("early,penalty", [(False, 1.0), (True, 1.0), (False, 0.0), (False, 2.0)])
def test_searches_follow_as_many_beams_as_they_can_whatever_ends(on_the_cpu, width, stops, early, penalty):
    """Against the definition, which looks at all continuations; at what ends, whatever that is, and at what goes on."""
    for seed in range(6):
        runner = PagedToy(seed)
        runner.table[..., list(stops)] += 1.0            # what ends is likely
        searcher = BeamSearcher(runner)
        searcher._select = select_by()
        params = BeamParams(width=width, max_tokens=9, length_penalty=penalty, early_stopping=early)
        prompts = [[2, 7], [5, 1, 0, 4, 12]]
        for prompt, found in zip(prompts, searcher.run(prompts, params, set(stops))):
            want = beam_search.search(runner.after, prompt, width, 9, penalty, early, set(stops))
            got = found.output().sequences
            assert [(s.output_token_ids, s.finish_reason.value) for s in got] == [(t, r) for t, _, _, r in want]
            assert all(abs(s.log_prob - p) < 1e-9 and abs(s.score - q) < 1e-9 for s, (_, p, q, _) in zip(got, want))
        empty(runner.cache)


def test_one_of_two_beams_is_looked_for_behind_what_ends():
    from kvforge_amd.engine.beams import Search
    s = Search([1], BeamParams(width=2, max_tokens=5), {8, 9}, 5)
    assert s.advance([(-1.0, 0, 3), (-1.1, 0, 4), (-3.0, 0, 8), (-4.0, 0, 9)]) == {0: 0, 1: 0}
    best = [(-1.2, 0, 5), (-1.3, 0, 9), (-1.4, 1, 9), (-1.5, 1, 8)]
    assert s.lacks(best, 4) and not s.lacks(best[:3], 4) and not s.lacks([*best[:2], (-1.4, 1, 5), best[3]], 4)
    assert s.advance(best, [best[0], (-4.0, 1, 0), (-4.1, 0, 0), (-4.2, 0, 1)]) == {0: 0, 1: 1}
    assert s.tokens == {0: [3, 5], 1: [4, 0]} and [e.output_token_ids for e in s.ended] == [[3, 9]] and not s.done
    # all of the best end: two have ended that no living one can pass
    ends = [(-2.2, 0, 8), (-2.3, 0, 9), (-2.4, 0, 6), (-2.5, 1, 8)]
    assert s.lacks(ends, 4)
    assert s.advance(ends, [ends[2], (-5.0, 1, 0)]) == {} and s.done


# ------------------------------------------------------------------------------------- searches that do not fit
@pytest.mark.parametrize("kind", ["pages", "slots", "positions", "empty"])
def test_a_list_of_prompts_is_refused_ahead_of_all_work(on_the_cpu, kind):
    """The last of them is the one that does not fit."""
    runner = PagedToy(blocks=16 if kind == "pages" else 120, seqs=3 if kind == "slots" else 16)
    runner.meta.max_seqs = 16
    searcher = BeamSearcher(runner)
    searcher._select = select_by()
    steps = []
    step = runner.step
    runner.step = lambda *a, **kw: (steps.append(1), step(*a, **kw))[1]
    last = {"pages": [1] * 50, "slots": [1, 2, 3], "positions": [1] * 64, "empty": []}[kind]
    params = BeamParams(width=4, max_tokens=5)
    with pytest.raises(ValueError):
        searcher.run([[1, 2], [3, 4, 5], last], params, set())
    assert not steps
    empty(runner.cache)
    if kind != "slots":
        assert all(s.done for s in searcher.run([[1, 2], [3, 4, 5]] * 3, params, set()))
        empty(runner.cache)


@pytest.mark.parametrize("seqs,tokens", [(16, 4), (16, 7), (16, 8), (4, 64), (9, 64)])
def test_batches_keep_to_the_sequences_and_tokens_of_a_step(on_the_cpu, seqs, tokens):
    runner = PagedToy(seqs=16, tokens=tokens)
    runner.meta.max_seqs = seqs
    searcher = BeamSearcher(runner)
    searcher._select = select_by()
    prompts = [[2, 7], [5, 1, 0, 4, 12], [3], [8, 8, 1, 2, 9, 10, 0, 4, 4, 4]]
    for prompt, found in zip(prompts, searcher.run(prompts, BeamParams(width=4, max_tokens=5), {3})):
        want = beam_search.search(runner.after, prompt, 4, 5, stops={3})
        assert [s.output_token_ids for s in found.output().sequences] == [t for t, _, _, _ in want]
    empty(runner.cache)
    with pytest.raises(ValueError):
        searcher.run(prompts, BeamParams(width=min(seqs, tokens) + 1, max_tokens=5), set())
    empty(runner.cache)
