"""Attention behind shared pages through an output gate: alone, where probabilities are powers of two and nothing but the one
rounding of the stored output is left, and in gated layers inside a search."""

from __future__ import annotations

import pytest
import torch

from tests.plain import beams as plain
from tests.test_beams import attend_args, launched  # noqa: F401
from tests.test_beams_gpu import DEV, paged

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32


def test_gates_that_are_refused(launched):  # noqa: F811
    from kvforge_amd.kernels import ops
    good = torch.zeros(4, 128)
    for gate in (good, torch.zeros(4, 300)[:, 100:228], torch.zeros(5, 128)):
        ops.attn_beams(**attend_args(), gate=gate)
    assert launched.count("kvf_attn_beams") == 3
    out = attend_args()
    for gate in (good.bfloat16(), torch.zeros(3, 128), torch.zeros(4, 127), torch.zeros(4, 256)[:, ::2], torch.zeros(4, 130)[:, :128],
                 torch.zeros(4, 132)[:, 1:129], out["out"]):
        with pytest.raises(ops.KernelError):
            ops.attn_beams(**out, gate=gate)
    assert launched.count("kvf_attn_beams") == 3


def gated(want, gate):
    return want / (1.0 + (-gate.detach().cpu().double()).exp())


def attend(q, k, v, tables, cu, shared, ctx, H, KV, d, scale, gate, sinks=None, cuts=(3, 2)):
    from kvforge_amd.kernels import ops
    n = len(ctx)
    ints = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    work = ops.attn_beams_workspace(n, H, d, cuts, DEV)
    out = torch.full((n, H * d), 7.0, dtype=k.dtype, device=DEV)
    ops.attn_beams(q.to(DEV), k.to(DEV), v.to(DEV), ints(tables), ints(cu), ints(shared), ints(ctx), out, H, KV, d, scale,
                   max(b - a for a, b in zip(cu, cu[1:])), cuts, work, sinks=sinks, gate=gate)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,KV,d,page,cuts", [(4, 2, 16, 16, (1, 1)), (6, 2, 80, 8, (3, 2)), (3, 3, 128, 16, (20, 20)), (8, 1, 256, 16, (2, 1)), (40, 2, 32, 3, (2, 2))])
def test_outputs_are_gated_ahead_of_their_one_rounding(dtype, H, KV, d, page, cuts):
    """Queries of zeros: every probability is one, ahead of the division.  32 bits: sums of up to 200 values are off by 200 2^-24 of
    their sizes at most, exponential and division by a few 2^-24: 2.5e-5 covers both.  bf16: one half step, 2^-8, beside it."""
    groups = [(96, [97, 130, 110]), (48, [48, 60]), (0, [0, 200]), (16, [17])]
    k, v, tables, cu, shared, ctx = paged(groups, KV, d, page, dtype, d)
    g = torch.Generator().manual_seed(d)
    wide = (torch.randn(len(ctx), H * d + 12, generator=g) * 4).to(dtype)
    wide[:, 8:20] = torch.tensor([-200.0, 200.0, 0.0, -90.0] * 3).to(dtype)
    gate = wide.to(DEV)[:, 8:8 + H * d]                                     # columns of a wider tensor
    out = attend(torch.zeros(len(ctx), H * d, dtype=dtype), k, v, tables, cu, shared, ctx, H, KV, d, 0.3, gate, cuts=cuts)
    want, weight = plain.attend(torch.zeros(len(ctx), H * d), k, v, tables, ctx, H, KV, d, 0.3)
    want, weight = gated(want, gate), gated(weight, gate)
    bound = 2.5e-5 * weight + 1e-30
    if dtype == BF16:
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    assert out[ctx.index(0)].eq(0).all()


@pytest.mark.gpu
def test_gates_beside_sinks_and_of_one_sequence():
    H, KV, d = 8, 2, 64
    k, v, tables, cu, shared, ctx = paged([(64, [90])], KV, d, 16, F32, 4)
    g = torch.Generator().manual_seed(2)
    q, gate, sinks = torch.randn(1, H * d, generator=g), torch.randn(1, H * d, generator=g), torch.randn(H, generator=g)
    out = attend(q, k, v, tables, cu, shared, ctx, H, KV, d, 0.125, gate.to(DEV), sinks.to(DEV))
    want, weight = plain.attend(q, k, v, tables, ctx, H, KV, d, 0.125, sinks)
    assert bool(((out.cpu().double() - gated(want, gate)).abs() <= 2.5e-5 * weight + 1e-7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_layers_inside_a_search(tmp_path_factory, monkeypatch, dtype):
    """Gated layers over all keys (this design's layers with their windows taken off) hand the gate to the kernel, which leaves no
    rounding and no launch behind it."""
    import kvforge_amd
    from kvforge_amd import BeamParams
    from kvforge_amd.engine.beams import BeamSearcher
    from kvforge_amd.engine.runner import ModelRunner
    from kvforge_amd.kernels import ops
    from kvforge_amd.models.transformer import Transformer
    from kvforge_amd.parts.attention import PagedAttention
    from tests import test_fogorax_gpu as fogorax
    cfg = fogorax.make_config(vocab=300, width=128, layers=2, heads=8, kv_heads=1, dim=64, ff=256, window=1000, keep_first=4, side_dim=64,
                              max_positions=900, share_every=1)
    folder = str(tmp_path_factory.mktemp("beams_gated"))
    kvforge_amd.write_random_model(folder, cfg, seed=12, dtype=fogorax.NAME[dtype])
    fogorax.liven(folder)
    init = PagedAttention.__init__

    def whole(self, *a, **kw):
        init(self, *a, **dict(kw, window=None, keep_first=0))
    monkeypatch.setattr(PagedAttention, "__init__", whole)
    runner = ModelRunner(Transformer.from_folder(folder, dtype, DEV), 16, 128, max_num_seqs=8, max_num_batched_tokens=512, max_model_len=900,
                         use_graphs=False)
    assert all(group.window is None for group in runner.cache.groups)
    real, sigmoid, seen = ops.attn_beams, ops.sigmoid_gate, []

    def checked(q, k, v, table, cu, shared, ctx, out, H, KV, d, scale, *rest, **kw):
        real(q, k, v, table, cu, shared, ctx, out, H, KV, d, scale, *rest, **kw)
        want, weight = plain.attend(q[:, :H * d], k, v, table.tolist(), ctx.tolist(), H, KV, d, scale)
        want, weight = gated(want, kw["gate"]), gated(weight, kw["gate"])
        bound = 2.5e-5 * weight + 1e-7
        if dtype == BF16:         # probabilities and the output, once each
            bound = bound + 2.0 ** -8 * weight + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -8)
        off = (out.cpu().double() - want).abs()
        assert bool((off <= bound).all()), float((off - bound).max())
        seen.append(len(ctx))
    gates: list = []
    monkeypatch.setattr(ops, "attn_beams", checked)
    monkeypatch.setattr(ops, "sigmoid_gate", lambda *a: (gates.append(a[0].shape[0]), sigmoid(*a)))
    prompts = [[(7 * i * i + n) % 300 for i in range(n)] for n in (600, 531)]
    found = BeamSearcher(runner).run(prompts, BeamParams(width=3, max_tokens=5), set())
    assert all(s.done for s in found) and len(seen) >= 8
    assert all(n > 8 for n in gates), "prompts only"
