"""Beam search over the step function and the paged cache.

A search keeps several continuations of a prompt, its beams, and each step of a batch of searches is: one forward over the
newest token of every living beam, ``ops.beam_select`` over the logits (the best ``2 * width`` continuations of every request;
with several stop tokens more than ``width`` of them may end, and the best of those that do not are selected by themselves where that
happens), and the beams' memory following the choice.  Pages that a beam has filled are shared by
its descendants (``CacheManager.branch``); the page that it is filling, and its state slots, are its own, and
``ops.beam_reorder`` copies them, in all layers with one launch a cache group.  A beam that goes on keeps its place (its
request id, rows and pages) with the first of its descendants, so only what has several is copied, into places whose beams were
not chosen.  Attention reads the pages that all beams of a request share, the prompt's above all, once (``ops.attn_beams``).

The reference has no beam search; names follow its sampling entry points (src/tokenvault/engine.py:105-194).
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import TYPE_CHECKING, Sequence

import numpy as np
import torch

from kvforge_amd.engine.batch import StepEntry
from kvforge_amd.engine.request import FinishReason
from kvforge_amd.kernels import ops
from kvforge_amd.sampling.params import BeamParams

if TYPE_CHECKING:  # pragma: no cover
    from kvforge_amd.engine.runner import ModelRunner


@dataclass
class BeamSequence:
    """One continuation: ``log_prob`` is the sum over its tokens, ``score`` what it is ranked by."""

    output_token_ids: list[int]
    log_prob: float
    score: float
    finish_reason: FinishReason
    text: str | None = None


@dataclass
class BeamOutput:
    prompt_token_ids: list[int]
    sequences: list[BeamSequence]


class Search:
    """The host's side of one request: its living beams by place (a place is a request id of the cache), and those that
    have ended."""

    def __init__(self, prompt: Sequence[int], params: BeamParams, stops: "set[int]", max_tokens: int) -> None:
        self.prompt, self.params, self.stops = list(prompt), params, stops
        self.max_tokens = max_tokens
        self.places: list[int] = [0]                # of the living beams, ascending
        self.tokens: dict[int, list[int]] = {0: []}
        self.log_probs: dict[int, float] = {0: 0.0}
        self.ended: list[BeamSequence] = []
        self.length = 0                             # output tokens of every living beam
        self.done = False

    def _end(self, tokens: list[int], log_prob: float, reason: FinishReason) -> None:
        self.ended.append(BeamSequence(tokens, log_prob, log_prob / len(tokens) ** self.params.length_penalty, reason))
        self.ended.sort(key=lambda s: -s.score)     # stable: of equals the first to end comes first
        del self.ended[self.params.width:]

    def lacks(self, candidates: "Sequence[tuple[float, int, int]]", asked: int) -> bool:
        """Whether so many of the ``asked`` best candidates end that there may be others to go on with behind them."""
        return len(candidates) >= asked and sum(token not in self.stops for _, _, token in candidates) < self.params.width

    def advance(self, candidates: "Sequence[tuple[float, int, int]]",
                going_on: "Sequence[tuple[float, int, int]] | None" = None) -> dict[int, int]:
        """Take the step's candidates (log-probability, number of the living beam, token), best first, and, where they lack such,
        the best of those that do not end.  Returns the parent's place of every living place; those whose beam goes on in its own
        place are their own parents."""
        width = self.params.width
        self.length += 1
        for log_prob, beam, token in candidates[:width]:        # what ends must be among the best itself
            if token in self.stops:
                self._end(self.tokens[self.places[beam]] + [token], log_prob, FinishReason.STOP)
        chosen = [(self.places[beam], token, log_prob) for log_prob, beam, token in (candidates if going_on is None else going_on)
                  if token not in self.stops][:width]
        if self.length >= self.max_tokens:
            for place, token, log_prob in chosen:
                self._end(self.tokens[place] + [token], log_prob, FinishReason.LENGTH)
            chosen = []
        elif chosen and len(self.ended) >= width:
            best = max(log_prob for _, _, log_prob in chosen) / self.length ** self.params.length_penalty
            if self.params.early_stopping or best <= self.ended[-1].score:
                chosen = []
        self.done = not chosen
        # the first descendant keeps its parent's place, the others take what is free
        kept = {place for place, _, _ in chosen}
        free = iter(p for p in range(width) if p not in kept)
        parents: dict[int, int] = {}
        tokens, log_probs = {}, {}
        for place, token, log_prob in chosen:
            to = place if place not in parents else next(free)
            parents[to] = place
            tokens[to], log_probs[to] = self.tokens[place] + [token], log_prob
        self.tokens, self.log_probs, self.places = tokens, log_probs, sorted(parents)
        return parents

    def output(self, tokenizer=None) -> BeamOutput:
        best = self.ended[:self.params.num_return or self.params.width]
        if tokenizer is not None:
            for s in best:
                s.text = tokenizer.decode(s.output_token_ids)
        return BeamOutput(self.prompt, best)


class BeamSearcher:
    """Runs searches on a ``ModelRunner`` beside whatever else holds pages there."""

    def __init__(self, runner: "ModelRunner") -> None:
        self.runner, self.cache, self.device = runner, runner.cache, runner.device
        storage = runner.storage
        # what beams own: the pages of every cache group, and the state slots, of all layers
        self.pages = [ops.CacheRows([t for layer in group.layers for t in storage.pages[layer].values()])
                      for group in self.cache.groups]
        states = list(runner.states.tensors.values())
        self.states = ops.CacheRows([t.flatten(1) for t in states]) if states else None
        self._kept: dict[tuple, tuple] = {}
        self._count = 0

    # ------------------------------------------------------------------ device work
    def _select(self, logits: torch.Tensor, searches: "list[Search]", count: int, ruled_out: torch.Tensor | None = None):
        """Candidates of every search, best first, as lists of (log-probability, beam, token)."""
        rows, vocab = logits.shape
        requests = len(searches)
        key = (rows, requests, count)
        if key not in self._kept:
            if len(self._kept) >= 64:
                del self._kept[next(iter(self._kept))]
            out = torch.empty(3, requests, count, dtype=torch.int32, device=self.device)
            ints = torch.zeros(rows + requests + 1, dtype=torch.int32, pin_memory=True)
            self._kept[key] = (out, ops.beam_select_workspace(rows, vocab, count, self.device), ints,
                               torch.empty_like(ints, device=self.device))
        out, work, host, dev = self._kept[key]
        flat = host.numpy()
        flat[:rows].view(np.float32)[:] = [s.log_probs[p] for s in searches for p in s.places]
        flat[rows] = 0
        flat[rows + 1:] = np.cumsum([len(s.places) for s in searches])
        dev.copy_(host, non_blocking=True)
        ops.beam_select(logits, dev[:rows].view(torch.float32), dev[rows:], out[0].view(torch.float32), out[1], out[2], work,
                        ruled_out)
        got = out.cpu().numpy()             # waits: the staging memory is free again
        scores, beams, tokens = got[0].view(np.float32).tolist(), got[1].tolist(), got[2].tolist()
        return [[c for c in zip(*request) if c[1] >= 0] for request in zip(scores, beams, tokens)]

    def _follow(self, searches: "list[Search]", ids: "list[list[str]]", parents: "list[dict[int, int]]", width: int) -> None:
        """The places' pages and slots become what their parents' were."""
        cache, bs = self.cache, self.cache.block_size
        moves = [(s, i, {to: p for to, p in by.items() if to != p}) for s, i, by in zip(searches, ids, parents)]
        partial = [(len(s.prompt) + s.length - 1) % bs != 0 for s in searches]       # whether a page is being filled
        for s, i, by in moves:
            for to, p in by.items():
                cache.branch(i[to], i[p], len(s.prompt) + s.length - 1)
        kinds = [*range(cache.num_groups), *([-1] if self.states is not None else [])]       # (-1: state slots)
        if not any(by for _, _, by in moves) or not kinds:
            return
        table = np.full((len(kinds), 2, len(searches), width), -1, dtype=np.int32)
        used = [False] * len(kinds)
        for r, (s, i, by) in enumerate(moves):
            for k, g in enumerate(kinds):
                if not by or (g >= 0 and not partial[r]):
                    continue
                used[k] = True
                for place in {*by, *by.values()}:
                    table[k, 0, r, place] = cache.slots.slot(i[place]) if g < 0 else cache.block_table(i[place], g)[-1]
                for to, p in by.items():
                    table[k, 1, r, to] = p
        if not any(used):
            return
        dev = torch.from_numpy(table).to(self.device)
        for k, g in enumerate(kinds):
            if used[k]:
                ops.beam_reorder(self.states if g < 0 else self.pages[g], dev[k, 0], dev[k, 1])

    # ------------------------------------------------------------------ searching
    def pages_needed(self, prompt_len: int, params: BeamParams, max_tokens: int) -> int:
        """Pages that a search can come to hold, a group: the prompt's once, and every beam's own behind those it fills."""
        bs = self.cache.block_size
        return prompt_len // bs + params.width * (-(-(prompt_len % bs + max_tokens) // bs))

    def run(self, prompts: "list[list[int]]", params: BeamParams, stops: "set[int]") -> "list[Search]":
        """Search all prompts, as many at a time as there is room for."""
        runner, cache = self.runner, self.cache
        searches, needs = [], []
        for prompt in prompts:
            if not prompt:
                raise ValueError("a beam search needs a prompt of at least one token")
            most = min(params.max_tokens, runner.max_model_len - len(prompt))
            if most < 1:
                raise ValueError(f"a prompt of {len(prompt)} tokens leaves no room for output within max_model_len "
                                 f"{runner.max_model_len}")
            searches.append(Search(prompt, params, stops, most))
            needs.append(self.pages_needed(len(prompt), params, most))
        at_once = min(runner.meta.max_seqs, runner.meta.max_tokens)        # beams of a step, a token each
        if params.width > at_once:
            raise ValueError(f"{params.width} beams are more than the {at_once} that a step takes ({runner.meta.max_seqs} sequences, "
                             f"{runner.meta.max_tokens} tokens)")
        # (a batch gives back what it held, so there is as much for each)
        free = min((p.num_free for p in cache.pools), default=math.inf)
        slots = cache.slots.num_free if cache.slots.num_slots else math.inf
        for s, need in zip(searches, needs):        # ahead of all work
            if need > free or params.width > slots:
                raise ValueError(f"a search of {params.width} beams behind {len(s.prompt)} tokens needs {need} pages and {params.width} state "
                                 f"slots, {free} pages and {slots} slots are free")
        at = 0
        while at < len(searches):
            n = pages = 0
            while (at + n < len(searches) and (n + 1) * params.width <= min(at_once, slots)
                   and pages + needs[at + n] <= free):
                pages += needs[at + n]
                n += 1
            self._run_batch(searches[at:at + n])
            at += n
        return searches

    def _run_batch(self, batch: "list[Search]") -> None:
        ids = []
        try:
            for s in batch:
                ids.append([f"beam-{self._count}-{p}" for p in range(s.params.width)])
                self._count += 1
                self.cache.allocate(ids[-1][0], len(s.prompt))
            self._search(batch, ids)
        finally:
            for request in ids:
                for rid in request:
                    self.cache.free(rid)

    def _read_prompts(self, batch: "list[Search]", ids: "list[list[str]]") -> torch.Tensor:
        """The prompts' tokens in portions; the logits behind each."""
        runner = self.runner
        logits = torch.empty(len(batch), runner.model.config.vocab_size, dtype=torch.float32, device=self.device)
        done = [0] * len(batch)
        while True:
            entries, rows, room = [], [], runner.meta.max_tokens
            for r, (s, i) in enumerate(zip(batch, ids)):
                n = min(len(s.prompt) - done[r], room)
                if n <= 0:
                    continue
                last = done[r] + n == len(s.prompt)
                entries.append(StepEntry(i[0], s.prompt[done[r]:done[r] + n], done[r], "last" if last else "none"))
                if last:
                    rows.append(r)
                done[r] += n
                room -= n
            if not entries:
                return logits
            found = runner.step(entries)
            if rows:
                logits[rows] = found
            for e in entries:
                self.cache.release_behind(e.request_id, e.start_pos + len(e.token_ids))

    @torch.inference_mode()
    def _search(self, batch: "list[Search]", ids: "list[list[str]]") -> None:
        cache, bs = self.cache, self.cache.block_size
        width = batch[0].params.width
        logits = self._read_prompts(batch, ids)
        common = [0] * len(batch)           # filled pages that all living beams of a search, and so their descendants, share
        living = list(range(len(batch)))
        ruled_out = None                    # the stop tokens, on the device (all searches have the same)
        while True:
            searches = [batch[r] for r in living]
            found = self._select(logits, searches, 2 * width)
            going_on = [None] * len(searches)
            lacking = [s.lacks(c, 2 * width) for s, c in zip(searches, found)]
            if any(lacking):
                if ruled_out is None:
                    stops = [t for t in sorted(batch[0].stops) if 0 <= t < logits.shape[1]]
                    ruled_out = torch.tensor(stops, dtype=torch.int32, device=self.device)
                others = self._select(logits, searches, 2 * width, ruled_out)
                going_on = [c if short else None for c, short in zip(others, lacking)]
            parents = [s.advance(c, o) for s, c, o in zip(searches, found, going_on)]
            self._follow(searches, [ids[r] for r in living], parents, width)
            for r in living:
                s = batch[r]
                for p, rid in enumerate(ids[r]):
                    if s.done or p not in s.tokens:
                        cache.free(rid)
            living = [r for r in living if not batch[r].done]
            if not living:
                return
            entries, shared = [], []
            for r in living:
                s = batch[r]
                pos = len(s.prompt) + s.length - 1
                here = [ids[r][p] for p in s.places]
                # (of one beam alone even the page that it fills is "shared", until it branches)
                common[r] = min(cache.shared_pages(here, common[r]), pos // bs)
                for p, rid in zip(s.places, here):
                    cache.append_slots(rid, pos + 1, pos)
                    entries.append(StepEntry(rid, [s.tokens[p][-1]], pos, "last"))
                shared.append((len(here), common[r] * bs))
            logits = self.runner.step(entries, shared=shared)
            for e in entries:
                cache.release_behind(e.request_id, e.start_pos + 1)
