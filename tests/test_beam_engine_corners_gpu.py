"""Beam search through the engine where a request has fewer continuations than beams."""
import pytest
import torch

from helpers import CONFIGS, make_model_folder
from test_beam_engine_gpu import compare, engine_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams,vocab", [(8, 6), (3, 2), (6, 1)])
def test_more_beams_than_tokens(tmp_path, beams, vocab):
    """Beams without a token keep rows in the steps, whatever their pages hold from earlier: the search is that of the definition."""
    config = dict(CONFIGS["D"][0], vocab_size=vocab)
    engine = engine_for(make_model_folder(str(tmp_path / "m"), config, 5))
    for g in engine.runner.cache.groups:
        g.storage.fill_(float("nan"))
    before = engine.generate([[0] * 9], max_new_tokens=4)
    for g in engine.runner.cache.groups:
        g.storage.zero_()
    assert engine.generate([[0] * 9], max_new_tokens=4) == before          # (prompts and steps do not read what they have not written)
    for g in engine.runner.cache.groups:
        g.storage.fill_(float("nan"))
    if vocab == 1:
        hyps, = engine.beam_search([[0] * 9], beams, 5, eos_tokens=[])
        assert [h.tokens for h in hyps] == [[0] * 5] and abs(hyps[0].score) <= 1e-5
    else:
        compare(engine, (9, 16, 21), beams, 5)
    assert all(torch.isfinite(torch.tensor([h.score for h in x])).all() for x in engine.beam_search([[0] * 3, [0] * 20], beams, 4, eos_tokens=[]))


def test_the_best_continuation_decides_whether_a_search_ends():
    """Two beams.  Once two have finished the search goes on while the step's best continuation is better than the worst of them, also where a stop token ends
    just that continuation and the best beam is worse than both."""
    from inferloop_b200.csrc import ops
    dev = "cuda:0"
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=dev)  # noqa: E731
    stops = torch.tensor([7], dtype=torch.int32, device=dev)

    def keep(track, step, tokens, scores):
        ops.beam_keep(i32([0, 0, 1, 1]), i32(tokens), torch.tensor([scores], device=dev), stops, track, step, 9, 0.0, False)
        return int(track.done), track.done_scores[0].tolist(), track.scores[0].tolist()
    a = ops.BeamTrack.make(1, 2, 9, dev)
    assert keep(a, 0, [1, 7, 2, 3], [-2.0, -3.0, -4.0, -5.0]) == (0, [-3.0, float("-inf")], [-2.0, -4.0])
    assert keep(a, 1, [7, 1, 2, 3], [-2.5, -3.5, -4.0, -5.0]) == (0, [-2.5, -3.0], [-3.5, -4.0])
    assert keep(a, 2, [1, 7, 2, 3], [-4.0, -4.5, -5.0, -6.0]) == (1, [-2.5, -3.0], [-4.0, -5.0])
    b = ops.BeamTrack.make(1, 2, 9, dev)
    assert keep(b, 0, [7, 1, 2, 3], [-1.0, -2.0, -3.0, -4.0]) == (0, [-1.0, float("-inf")], [-2.0, -3.0])
    assert keep(b, 1, [7, 1, 2, 3], [-2.5, -3.5, -4.0, -5.0]) == (1, [-1.0, -2.5], [-3.5, -4.0])      # (no better than the worst, which it is)
