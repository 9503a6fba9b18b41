"""What the command line takes beside ``--beams``."""

from __future__ import annotations

import pytest

from kvforge_amd import generate


@pytest.mark.parametrize("args", [["--beams", "4"], ["--beams", "1", "--length-penalty", "0.5", "--early-stopping"], ["--beams", "32", "--seed", "3"],
                                  ["--beams", "2", "--temperature", "0", "--top-k", "0", "--top-p", "1"], ["--temperature", "0.7", "--seed", "3"],
                                  ["--model", "DIR", "--beams", "2"], ["--model", "DIR", "--seed", "2"]])
def test_taken(args):
    said = generate.parse_args(args)
    assert said.beams is None or generate._beam_params(said).width == said.beams


@pytest.mark.parametrize("args,why", [(["--beams", "0"], "1 to 32 beams"), (["--beams", "33"], "1 to 32 beams"), (["--beams", "-1"], "1 to 32 beams"),
                                      (["--beams", "2", "--max-tokens", "0"], "max_tokens"), (["--beams", "2", "--temperature", "0.7"], "--temperature"),
                                      (["--beams", "2", "--top-k", "5"], "--top-k"), (["--beams", "2", "--top-p", "0.9"], "--top-p"),
                                      (["--beams", "2", "--model", "DIR", "--seed", "1"], "--seed"), (["--length-penalty", "2"], "--beams"),
                                      (["--early-stopping"], "--beams")])
def test_refused_in_words(args, why, capsys):
    with pytest.raises(SystemExit) as ended:
        generate.parse_args(args)
    assert ended.value.code == 2 and why in capsys.readouterr().err
