"""Selection without tokens that the caller rules out: refusals on the CPU; on the GPU against the plain form, whose scores stay those
of all tokens, and whole searches with several stop tokens against their definition."""

from __future__ import annotations

import math

import pytest
import torch

from kvforge_amd import BeamParams
from tests.plain import beam_search, beams as plain
from tests.test_beams import launched, select_args  # noqa: F401

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
DEV = "cuda"


def test_what_may_be_ruled_out(launched):  # noqa: F811
    from kvforge_amd.kernels import ops
    for good in (torch.tensor([3, 5], dtype=I32), torch.zeros(0, dtype=I32), None):
        ops.beam_select(**select_args(), ruled_out=good)
    assert launched == ["kvf_beam_select"] * 3
    for bad in (torch.tensor([3, 5]), torch.zeros(2, 1, dtype=I32), torch.zeros(4, dtype=I32)[::2], torch.zeros(2)):
        with pytest.raises(ops.KernelError):
            ops.beam_select(**select_args(), ruled_out=bad)
    args = select_args()
    with pytest.raises(ops.KernelError):
        ops.beam_select(**args, ruled_out=args["out_tokens"].view(-1))
    assert len(launched) == 3


def select(logits, scores, cu, count, ruled=None):
    from kvforge_amd.kernels import ops
    ints = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    shape = (len(cu) - 1, count)
    outs = (torch.full(shape, 7.0, device=DEV), torch.full(shape, 7, dtype=I32, device=DEV), torch.full(shape, 7, dtype=I32, device=DEV))
    ops.beam_select(logits, scores, ints(cu), *outs, ops.beam_select_workspace(*logits.shape, count, DEV),
                    **({} if ruled is None else {"ruled_out": ints(ruled)}))
    return outs


def rest_of(logits, scores, cu, count, ruled):
    """What all candidates come to without those that are ruled out."""
    out = set(ruled)
    return [[c for c in found if c[2] not in out][:count] for found in plain.select(logits, scores, cu, logits.shape[0] * logits.shape[1])]


def ruled_lists(vocab, piece=2048):
    edges = [t for p in range(0, vocab, piece) for t in (p - 9, p - 8, p - 1, p, p + 1, p + 7)]
    return {"none": [], "one": [vocab // 2], "edges": edges + [vocab - 1, vocab, vocab + 5, -1, -2**31, 2**31 - 1], "all": list(range(vocab)),
            "twice": [0, 0, 1, 0], "all but two": [t for t in range(vocab) if t not in (vocab // 3, vocab - 1)][::-1]}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "one", "edges", "all", "twice", "all but two"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,beams,count,offset", [(1, 1, 1, 1, 0), (4, 70, 2, 8, 1), (6, 2047, 3, 6, 0), (5, 2049, 5, 33, 3), (8, 5003, 4, 64, 5),
                                                         (12, 9001, 4, 24, 2)])
def test_selection_without_what_is_ruled_out(kind, dtype, rows, vocab, beams, count, offset):
    g = torch.Generator().manual_seed(rows * vocab)
    ruled = ruled_lists(vocab)[kind]
    wide = torch.full((rows, vocab + 16), 99.0).to(dtype)
    logits = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    logits[:, [t for t in ruled if 0 <= t < vocab][:50]] += 4.0          # what is ruled out is large
    wide[:, offset:offset + vocab] = logits
    held = wide.to(DEV)[:, offset:offset + vocab]
    scores = -torch.rand(rows, generator=g) * 5
    cu = list(range(0, rows, beams)) + [rows]
    got_s, got_b, got_t = (t.cpu() for t in select(held, scores.to(DEV), cu, count, ruled))
    for r, expected in enumerate(rest_of(logits, scores, cu, count, ruled)):
        n = len(expected)
        assert got_b[r, n:].eq(-1).all() and got_t[r, n:].eq(-1).all() and got_s[r, n:].eq(-math.inf).all()
        for i, (s, b, t) in enumerate(expected):
            # (a sum is off by a few 2^-24: 2^-21; scores of two beams that near may change places)
            assert abs(float(got_s[r, i]) - s) <= 2.0 ** -24 * abs(s) + 2.0 ** -21
            if not any(abs(x[0] - s) <= 2.0 ** -20 and x[1] != b for x in expected):
                assert (int(got_b[r, i]), int(got_t[r, i])) == (b, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(8, 3000), (40, 40001)])
def test_scores_are_those_of_a_call_that_rules_out_nothing(dtype, rows, vocab):
    """To the bit, with NaN, infinities and dead beams: both calls select everything that is left, in the same order."""
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 2)
    logits[1], logits[2, ::2], logits[3, 7] = math.nan, -math.inf, math.inf
    scores = -torch.rand(rows, generator=g)
    scores[5] = -math.inf
    logits, scores, cu = logits.to(dtype).to(DEV), scores.to(DEV), list(range(0, rows + 1, 4))
    every = [list(zip(*x)) for x in zip(*(t.tolist() for t in select(logits, scores, cu, 64)))]
    ruled = sorted({c[2] for found in every for c in found[:20:2]} - {-1})
    some = [list(zip(*x)) for x in zip(*(t.tolist() for t in select(logits, scores, cu, 64, ruled)))]
    for a, b in zip(every, some):
        left = [c for c in a if c[2] not in ruled]
        assert b[:len(left)] == left and not any(c[2] in ruled for c in b)


@pytest.mark.gpu
@pytest.mark.parametrize("width,many", [(2, 40), (4, 25), (4, 120), (5, 254), (3, 255)])
@pytest.mark.parametrize("graphs", [True, False])
def test_searches_with_many_stop_tokens_are_the_definition(tmp_path_factory, width, many, graphs):
    """Sequences are those of the definition where none of its choices goes by less than 1e-4 (32-bit logits are off by less than 4e-6, sums of a
    dozen log-probabilities by less than 1e-4)."""
    from tests.test_beam_search_gpu import empty, engine_for, llama_model, prompts_of, remembered
    folder, logits = llama_model(tmp_path_factory, "tiny-a", 0)
    ask = remembered(logits)
    stops = torch.randperm(256, generator=torch.Generator().manual_seed(many))[:many].tolist()
    engine = engine_for(folder, block=4, use_graphs=graphs)
    asked, strict = [], 0
    from kvforge_amd.kernels import ops
    real = ops.beam_select
    ops.beam_select = lambda *a, **kw: (asked.append(a[-1] is not None), real(*a, **kw))
    try:
        prompts = prompts_of(256, [3, 8, 21, 34, 5, 6], seed=width)
        for penalty, early in ((1.0, False), (0.0, False), (2.0, True)):
            params = BeamParams(width=width, max_tokens=10, length_penalty=penalty, early_stopping=early, stop_token_ids=stops, ignore_eos=False)
            ends = {*stops, *([] if engine.model.config.eos_token_id is None else [engine.model.config.eos_token_id])}
            for prompt, out in zip(prompts, engine.beam_search(prompts, params)):
                gaps: list = []
                want = beam_search.search(ask, prompt, width, 10, penalty, early, ends, gaps)
                assert all(math.isfinite(s.log_prob) for s in out.sequences) and len(out.sequences) == len(want)
                if min(gaps, default=1.0) > 1e-4:
                    strict += 1
                    assert [(s.output_token_ids, s.finish_reason.value) for s in out.sequences] == [(t, r) for t, _, _, r in want]
                    assert all(abs(s.score - q) < 1e-4 for s, (_, _, q, _) in zip(out.sequences, want))
            empty(engine)
    finally:
        ops.beam_select = real
    assert strict >= 9 and (many < 100 or any(asked))
