"""What beams read behind shared pages while a search narrows to one beam and widens again: the engine's searches against the
plain models, and attention inside the steps against the plain form over the same pages."""

from __future__ import annotations

import pytest
import torch

from kvforge_amd import BeamParams
from tests.plain import beams as plain
from tests.test_beam_search_gpu import empty, engine_for, llama_model, prompts_of, remembered

pytestmark = pytest.mark.gpu


def narrowed(engine, lives):
    """The engine's searcher, whose ``n``-th selection leaves only ``lives[n]`` of a request's candidates."""
    from kvforge_amd.engine.beams import BeamSearcher
    engine._beams = searcher = BeamSearcher(engine.runner)
    select, turns = searcher._select, []

    def few(*args):
        turns.append(len(turns))
        return [found[:lives[turns[-1] % len(lives)]] for found in select(*args)]
    searcher._select = few
    return engine


@pytest.mark.parametrize("graphs", [True, False])
def test_searches_that_narrow_to_one_beam_and_widen(tmp_path_factory, graphs):
    """32 bits, where any shared key takes the shared kernel: log-probabilities are those of the tokens (the engine's logits are off
    by less than 4e-6, sums over a dozen tokens by less than 1e-4)."""
    folder, logits = llama_model(tmp_path_factory, "tiny-a", 0)
    ask, prompts = remembered(logits), prompts_of(256, [5, 18, 39], seed=11)
    for lives in ((4, 1, 3, 3), (1, 1, 4, 2, 1)):
        engine = narrowed(engine_for(folder, block=4, use_graphs=graphs), lives)
        for prompt, out in zip(prompts, engine.beam_search(prompts, BeamParams(width=4, max_tokens=12))):
            assert out.sequences
            for s in out.sequences:
                total = sum(float(torch.log_softmax(ask(prompt + s.output_token_ids[:i]).double(), dim=0)[t])
                            for i, t in enumerate(s.output_token_ids))
                assert abs(s.log_prob - total) < 1e-4, (lives, len(prompt), s.output_token_ids)
        empty(engine)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_inside_the_steps_of_a_search(tmp_path_factory, dtype):
    """Every layer's attention of every step, from the pages as they then are, every sequence's keys looked up in its own table.  A
    score is off by 2^-24 sqrt(d) of its size and probabilities by as much: 2.5e-5 of the sum of |p v| covers it (scores up
    to 8).  bf16 adds the rounding of probabilities, 2^-8 of that sum, and of the stored output, 2^-8 of it."""
    import kvforge_amd
    from kvforge_amd.kernels import ops
    from tests.replay_util import liven
    cfg = dict(kvforge_amd.preset_dict("tiny-b"), head_dim=64, num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=2048)
    folder = str(tmp_path_factory.mktemp("beams_inside"))
    kvforge_amd.write_random_model(folder, cfg, seed=2, dtype=dtype)
    liven(folder)
    engine = narrowed(engine_for(folder, dtype, block=16, tokens=512, seqs=8, use_graphs=False), (4, 1, 3, 2))
    real, seen = ops.attn_beams, []

    def checked(q, k, v, table, cu, shared, ctx, out, H, KV, d, scale, *rest, **kw):
        real(q, k, v, table, cu, shared, ctx, out, H, KV, d, scale, *rest, **kw)
        lens = ctx.tolist()
        want, weight = plain.attend(q[:, :H * d], k, v, table.tolist(), lens, H, KV, d, scale)
        bound = 2.5e-5 * weight + 1e-7
        if out.dtype == torch.bfloat16:
            bound = bound + 2.0 ** -8 * weight + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8)
        off = (out.cpu().double() - want).abs()
        assert bool((off <= bound).all()), (len(seen), lens, float((off - bound).max()))
        seen.append(len(lens))
    ops.attn_beams = checked
    try:
        engine.beam_search(prompts_of(384, [531, 700], seed=5), BeamParams(width=4, max_tokens=10))
    finally:
        ops.attn_beams = real
    assert {2, 6, 8} <= set(seen)          # one beam a prompt, three, four
