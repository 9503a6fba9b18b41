"""Beam search through the engine against its definition over the plain models: paged attention alone, windows with
recurrent states and routed experts, latent pages with short convolutions and delta memories; prompts of unequal lengths in
several batches, stop tokens, pages that beams share and those they fill, captured steps, and the command line."""

from __future__ import annotations

import json
import math
import random

import pytest
import torch

import kvforge_amd
from kvforge_amd import BeamParams, EngineConfig, InferenceEngine, SamplingParams
from kvforge_amd.config.engine import CacheConfig, SchedulerConfig
from tests.plain import beams as plain
from tests.plain import depolix as plain_depolix
from tests.plain import llama as plain_llama
from tests.plain import rudorax as plain_rudorax

pytestmark = pytest.mark.gpu


def llama_model(tmp_path_factory, preset, seed, dtype="float32", liven=True):
    from tests.replay_util import liven as make_alive
    folder = str(tmp_path_factory.mktemp(f"beams_{preset}"))
    kvforge_amd.write_random_model(folder, kvforge_amd.preset_dict(preset), seed=seed, dtype=dtype)
    if liven:
        make_alive(folder)
    w, cfg = plain_llama.read_weights(folder), plain_llama.read_config(folder)
    return folder, lambda tokens: plain_llama.forward(w, cfg, tokens, dtype=torch.float64, last=1)[-1]


@pytest.fixture(scope="module")
def tiny_a(tmp_path_factory):
    return llama_model(tmp_path_factory, "tiny-a", 0)


@pytest.fixture(scope="module")
def tiny_b(tmp_path_factory):
    return llama_model(tmp_path_factory, "tiny-b", 1)


def remembered(logits):
    known: dict[tuple, torch.Tensor] = {}

    def ask(tokens):
        key = tuple(tokens)
        if key not in known:
            known[key] = logits(tokens)
        return known[key]
    return ask


def engine_for(folder, dtype="float32", block=4, blocks=256, seqs=16, tokens=64, **kw):
    return InferenceEngine.from_folder(folder, EngineConfig(
        cache=CacheConfig(block_size=block, num_blocks=blocks),
        scheduler=SchedulerConfig(max_num_seqs=seqs, max_num_batched_tokens=tokens), dtype=dtype, **kw))


def prompts_of(vocab, lengths, seed=0):
    rng = random.Random(seed)
    return [[rng.randrange(vocab) for _ in range(n)] for n in lengths]


def empty(engine):
    cache = engine.cache
    assert all(p.num_free == p.num_blocks for p in cache.pools)
    assert not cache.slots.num_slots or cache.slots.num_free == cache.slots.num_slots


def check(engine, logits, prompts, params, stops=(), off=1e-4):
    """Sequences are those of the definition where none of its choices goes by a difference below ``off`` (the
    engine's logits are off by less than 4e-6 in 32 bits, their log-softmax by twice that, sums of up to a dozen by less than it); every
    log-probability is that of its tokens.  Returns how many prompts were compared token by token."""
    ask = remembered(logits)
    strict = 0
    for prompt, out in zip(prompts, engine.beam_search(prompts, params)):
        most = min(params.max_tokens, engine.runner.max_model_len - len(prompt))
        want, gap = plain.search(ask, prompt, params.width, most, params.length_penalty, params.early_stopping, set(stops))
        assert out.prompt_token_ids == prompt and len(out.sequences) <= params.width
        for s in out.sequences:
            total = 0.0
            for i, t in enumerate(s.output_token_ids):
                total += float(torch.log_softmax(ask(prompt + s.output_token_ids[:i]).double(), dim=0)[t])
            assert abs(s.log_prob - total) < off and abs(s.score - s.log_prob / len(s.output_token_ids) ** params.length_penalty) < 1e-6
            assert (s.finish_reason.value == "stop") == (s.output_token_ids[-1] in stops)
        if gap > off:
            strict += 1
            assert [s.output_token_ids for s in out.sequences] == [t for t, _, _, _ in want], (prompt, gap)
            assert all(abs(s.score - q) < off for s, (_, _, q, _) in zip(out.sequences, want))
    empty(engine)
    return strict


@pytest.mark.parametrize("width", [1, 2, 4, 7])
def test_searches_are_the_definition(tiny_a, width):
    """Prompts around the page size of four, the long one in portions; nine searches in batches of what sixteen sequences hold."""
    folder, logits = tiny_a
    engine = engine_for(folder)
    prompts = prompts_of(256, [1, 3, 4, 5, 8, 21, 90, 12, 7], seed=width)
    assert check(engine, logits, prompts, BeamParams(width=width, max_tokens=10)) >= (3 if width == 7 else 7)


@pytest.mark.parametrize("early,penalty", [(False, 1.0), (True, 1.0), (False, 0.0), (True, 2.0)])
def test_searches_that_end_at_stop_tokens(tiny_b, early, penalty):
    folder, logits = tiny_b
    engine = engine_for(folder, block=8)
    stops = list(range(0, 384, 9))
    prompts = prompts_of(384, [5, 16, 33], seed=3)
    params = BeamParams(width=3, max_tokens=12, length_penalty=penalty, early_stopping=early, stop_token_ids=stops)
    eos = engine.model.config.eos_token_id
    assert check(engine, logits, prompts, params, [*stops, *([] if eos is None else [eos])]) >= 2
    ignored = BeamParams(width=3, max_tokens=6, stop_token_ids=stops, ignore_eos=True)
    assert check(engine, logits, prompts, ignored) >= 2


def test_one_beam_is_greedy(tiny_a):
    folder, _ = tiny_a
    engine = engine_for(folder)
    prompts = prompts_of(256, [6, 17], seed=9)
    greedy = engine.generate(prompts, SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True))
    found = engine.beam_search(prompts, BeamParams(width=1, max_tokens=12, ignore_eos=True))
    assert [o.output_token_ids for o in greedy] == [o.sequences[0].output_token_ids for o in found]
    empty(engine)


def test_searches_beside_requests_that_wait(tiny_a):
    """Requests under way keep their pages, and go on afterwards as if nothing had been."""
    folder, logits = tiny_a
    engine = engine_for(folder, blocks=64)
    alone = engine.generate(prompts_of(256, [9], seed=1), SamplingParams(max_tokens=12, temperature=0.0))
    engine.add_request(prompts_of(256, [9], seed=1)[0], SamplingParams(max_tokens=12, temperature=0.0))
    engine.step()
    used = engine.cache.stats().num_used_blocks
    found = engine.beam_search(prompts_of(256, [7], seed=2), BeamParams(width=4, max_tokens=6))
    assert engine.cache.stats().num_used_blocks == used
    want, _ = plain.search(logits, found[0].prompt_token_ids, 4, 6)
    assert found[0].sequences[0].output_token_ids == want[0][0]
    outs = []
    while engine.has_unfinished_requests():
        outs = engine.step()
    assert outs[-1].output_token_ids == alone[0].output_token_ids
    empty(engine)


def test_searches_that_do_not_fit_are_refused(tiny_a):
    folder, _ = tiny_a
    engine = engine_for(folder, blocks=12, seqs=4)
    for prompts, params in (([[1] * 40], BeamParams(width=4, max_tokens=8)), ([[1, 2]], BeamParams(width=5)), ([[]], BeamParams()),
                            ([[1, 999]], BeamParams())):
        with pytest.raises(ValueError):
            engine.beam_search(prompts, params)
        empty(engine)
    limit = engine.runner.max_model_len
    with pytest.raises(ValueError, match="no room"):
        engine.beam_search([[1] * limit], BeamParams(width=1))
    assert engine.beam_search([], BeamParams()) == []


def test_a_search_that_fails_gives_its_pages_back(tiny_a, monkeypatch):
    folder, _ = tiny_a
    engine = engine_for(folder)
    step, calls = engine.runner.step, []

    def failing(*a, **kw):
        calls.append(1)
        if len(calls) == 4:
            raise RuntimeError("stopped")
        return step(*a, **kw)
    monkeypatch.setattr(engine.runner, "step", failing)
    with pytest.raises(RuntimeError, match="stopped"):
        engine.beam_search(prompts_of(256, [5, 9]), BeamParams(width=3, max_tokens=9))
    empty(engine)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_shared_prompts_are_read_once_and_say_the_same(tmp_path_factory, dtype, graphs):
    """Behind prompts longer than what the shared kernel is taken from; the same search with every sequence's keys read by
    themselves.  Steps are captured and replayed while beams branch, end and cross page borders."""
    cfg = dict(kvforge_amd.preset_dict("tiny-b"), head_dim=64, num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=2048)
    folder = str(tmp_path_factory.mktemp("beams_long"))
    kvforge_amd.write_random_model(folder, cfg, seed=2, dtype=dtype)
    from tests.replay_util import liven
    liven(folder)
    w = plain_llama.read_weights(folder)
    logits = remembered(lambda tokens: plain_llama.forward(w, cfg, tokens, dtype=torch.float64, last=1)[-1])
    prompts = prompts_of(384, [700, 1100], seed=5)
    params = BeamParams(width=4, max_tokens=24)
    engine = engine_for(folder, dtype, block=16, tokens=512, seqs=8, use_graphs=graphs)
    calls = []
    from kvforge_amd.kernels import ops
    real = ops.attn_beams
    ops.attn_beams = lambda *a, **kw: (calls.append(a[4].shape[0] - 1), real(*a, **kw))
    try:
        found = engine.beam_search(prompts, params)
    finally:
        ops.attn_beams = real
    assert calls and set(calls) == {2}
    assert not graphs or engine.runner.num_graph_replays >= 8
    empty(engine)
    off = 1e-3 if dtype == "float32" else 0.5
    for prompt, out in zip(prompts, found):
        s = out.sequences[0]
        total = sum(float(torch.log_softmax(logits(prompt + s.output_token_ids[:i]).double(), dim=0)[t])
                    for i, t in enumerate(s.output_token_ids))
        assert abs(s.log_prob - total) < off, (s.log_prob, total)
    if dtype == "float32":
        apart = engine_for(folder, dtype, block=16, tokens=512, seqs=8, use_graphs=graphs)
        step = apart.runner.step
        apart.runner.step = lambda entries, shared=None: step(entries)
        assert [[s.output_token_ids for s in o.sequences] for o in apart.beam_search(prompts, params)] == \
            [[s.output_token_ids for s in o.sequences] for o in found]


def test_states_windows_and_experts_follow_their_beams(tmp_path_factory):
    """Matrix memories beside windowed attention: slots are copied, pages behind the window are given back."""
    from tests import test_rudorax_gpu as rudorax
    for shape in ("a", "c"):
        folder, cfg, w = rudorax.model_folder(tmp_path_factory, shape, torch.float32)
        logits = lambda tokens: plain_rudorax.forward(cfg, w, tokens, dtype=torch.float64)[-1]
        vocab = w["embed"].shape[0]
        engine = engine_for(folder, block=8, seqs=8)
        assert check(engine, logits, prompts_of(vocab, [3, 8, 41], seed=4), BeamParams(width=3, max_tokens=9), off=3e-4) >= 2


def test_latents_convolutions_and_delta_memories_follow_their_beams(tmp_path_factory):
    from safetensors.torch import load_file
    from tests import test_depolix_gpu as depolix
    cfg = depolix.shape_b()
    folder = str(tmp_path_factory.mktemp("beams_depolix"))
    kvforge_amd.write_random_model(folder, cfg, seed=7, dtype="float32")
    depolix.liven(folder, cfg)
    w = load_file(f"{folder}/model.safetensors")
    logits = lambda tokens: plain_depolix.forward(cfg, w, tokens, dtype=torch.float64)[-1]
    engine = engine_for(folder, block=4, seqs=8)
    assert check(engine, logits, prompts_of(w["embed"].shape[0], [2, 9, 30], seed=6), BeamParams(width=4, max_tokens=8), off=3e-4) >= 1


def test_the_command_line_searches(capsys):
    from kvforge_amd import generate
    args = ["--preset", "tiny-a", "--prompt-ids", "5,17,3", "--max-tokens", "5", "--beams", "3", "--num-blocks", "64"]
    assert generate.main([*args, "--json"]) == 0
    said = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    sequences = said["outputs"][0]["sequences"]
    assert len(sequences) == 3 and [s["score"] for s in sequences] == sorted((s["score"] for s in sequences), reverse=True)
    assert all(math.isfinite(s["log_prob"]) for s in sequences)
    assert generate.main(args) == 0
    assert "beams=3" in capsys.readouterr().out
