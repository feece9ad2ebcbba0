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
