"""A workspace of selection serves every smaller call: fewer rows, which may be cut into more pieces each."""

from __future__ import annotations

import pytest
import torch

from kvforge_amd.kernels import ops
from tests.test_beams import launched  # noqa: F401


@pytest.mark.parametrize("vocab,count", [(40, 4), (8192, 8), (50001, 24), (128256, 8), (128256, 64)])
def test_fewer_rows_fit_into_the_workspace_of_more(launched, vocab, count):  # noqa: F811
    made, ints = 0, lambda *shape: torch.zeros(*shape, dtype=torch.int32)
    for most in (1, 3, 16, 40, 63, 150, 600):
        work = ops.beam_select_workspace(most, vocab, count, "cpu")
        for rows in range(1, most + 1, 1 if most < 100 else 29):
            ops.beam_select(torch.empty(rows, vocab, dtype=torch.bfloat16), torch.zeros(rows), ints(2), torch.zeros(1, count), ints(1, count),
                            ints(1, count), work)
            made += 1
    assert launched == ["kvf_beam_select"] * made
