"""`infer generate --beams` with a stand-in for the engine: what it is given, what is printed, what is refused."""
import json

import pytest

from inferloop_b200 import BeamHypothesis, cli


@pytest.fixture
def asked(monkeypatch):
    calls = []

    class Engine:
        def beam_search(self, *args):
            calls.append(args)
            return [[BeamHypothesis([4, 9], -0.5, "eos"), BeamHypothesis([4, 8, 1], -0.75, "length")]]
    monkeypatch.setattr(cli, "_engine", lambda args, folder: calls.append(folder) or Engine())
    return calls


def generate(*options):
    args = cli.build_parser().parse_args(["generate", "folder", "--tokens", "5, 17,3", *options])
    return cli.cmd_generate(args)


@pytest.mark.parametrize("options,want", [
    (["--beams", "2"], (2, None, 1.0, False, None)),
    (["--beams", "4", "--max-new-tokens", "9", "--length-penalty", "0.5"], (4, 9, 0.5, False, None)),
    (["--beams", "1", "--early-stopping", "--eos-token", "7", "--length-penalty", "-2"], (1, None, -2.0, True, [7]))])
def test_options_reach_the_search(asked, capsys, options, want):
    assert generate(*options) == 0
    folder, (prompts, beams, last, penalty, early, stops) = asked
    default = cli.build_parser().parse_args(["generate", "m", "--tokens", "1"]).max_new_tokens
    assert folder == "folder" and prompts == [[5, 17, 3]]
    assert (beams, last, penalty, early, stops) == (want[0], default if want[1] is None else want[1], *want[2:])
    assert json.loads(capsys.readouterr().out) == {"beams": [{"tokens": [4, 9], "score": -0.5, "reason": "eos"},
                                                            {"tokens": [4, 8, 1], "score": -0.75, "reason": "length"}]}


@pytest.mark.parametrize("option", ["--temperature", "--top-k", "--top-p", "--min-p", "--presence-penalty", "--repetition-penalty", "--seed"])
def test_sampling_options_are_refused(asked, option):
    with pytest.raises(ValueError, match=option):
        generate("--beams", "2", option, "1")
    assert asked == []                                   # (before a model is loaded)
