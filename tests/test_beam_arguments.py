"""Arguments that the beam search cannot serve: refused before anything runs."""
from types import SimpleNamespace

import pytest
import torch

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


def test_storages_whose_heads_are_too_long(monkeypatch):
    """Without a device: storages of no memory, of which only shapes are looked at.  2^31 - 4096 bytes of a page's head is the most."""
    from inferloop_b200.csrc import ops
    monkeypatch.setattr(ops, "_need", lambda *a, **k: None)
    monkeypatch.setattr(ops, "_sm_count", lambda device: 1)
    cpu = torch.device("cpu")

    def make(rows, row, unit=1):
        x = SimpleNamespace(dim=lambda: 4, shape=(2, 1, rows, row), element_size=lambda: 1, numel=lambda: 2 * rows * row, data_ptr=lambda: 4096, device=cpu)
        return ops.BeamState([([x], rows * unit, 1)], [], cpu)
    for rows, row, unit in ((16, (1 << 27) - 256, 1), (4, (1 << 29) - 1024, 16), (1, (1 << 31) - 4096, 16)):
        assert make(rows, row, unit).parts == 1
    for rows, row, unit in ((16, 1 << 27, 1), (1 << 16, 1 << 15, 1), (4, (1 << 29) - 1023, 16), (1, (1 << 31) - 1, 16)):
        with pytest.raises(ops.KernelError, match="too long"):
            make(rows, row, unit)
