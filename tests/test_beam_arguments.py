"""Arguments of a beam search that no score could be told apart with: refused before anything runs."""
import pytest

from inferloop_b200.parts.base import CacheNeeds, PagedKVNeed
from test_beam_engine import search
from inferloop_b200.engine.beams import BeamSearch


@pytest.mark.parametrize("last,penalty,served", [(16, 25.0, True), (16, -25.0, True), (16, 25.5, False), (16, -30.0, False), (1, 1e6, True), (300, 12.0, True),
                                                 (300, 12.5, False), (4, float("inf"), False), (4, float("nan"), False)])
def test_length_penalties(last, penalty, served):
    s, _ = search([CacheNeeds(paged=PagedKVNeed(1, 16))], 4, 16, 4, 2, last)
    if served:
        assert BeamSearch(s.engine, 2, last, (), penalty).penalty == penalty
    else:
        with pytest.raises(ValueError):
            BeamSearch(s.engine, 2, last, (), penalty)
