"""How many recorded steps of beam searches are kept."""
from types import SimpleNamespace

import pytest
import torch

from helpers import CONFIGS, make_model_folder, random_tokens
from inferloop_b200.engine import graphs
from inferloop_b200.engine.graphs import DecodeGraphs, _Recorded


class Runner(SimpleNamespace):
    """(one that a weak reference can be taken of)"""


def beam_keys(g):
    return [k for k in g._recorded if k[0] == "beams"]


def test_the_latest_used_are_kept(monkeypatch):
    """Without a device: a stand-in for the recording, which is kept as a recording is."""
    synced = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(synchronize=lambda: synced.append(1)))
    monkeypatch.setattr(graphs, "BEAM_STEPS_KEPT", 3, raising=False)
    runner = Runner(model=SimpleNamespace(blocks=[SimpleNamespace(graph_safe=True)], graph_safe=True), device=torch.device("cpu"),
                    spec=SimpleNamespace(run_order=[SimpleNamespace(layer=0)], token_extras=(), max_positions=4096),
                    cache=SimpleNamespace(groups=[0]), ctx=SimpleNamespace(workspace=SimpleNamespace(generation=1)))
    g = DecodeGraphs(runner, 8)

    def search(rows, longest):
        key, rec, ctx, ints = g.beam_step(rows, 2, longest)
        if rec is None:
            g._recorded[key] = _Recorded([("graph", None)], ints, ctx, None, runner.ctx.workspace.generation, 0)
        return key, rec is not None
    g._recorded[4, True, False] = decode = _Recorded([("graph", None)], None, None, None, 1, 0)
    keys = [search(4, n)[0] for n in (64, 128, 256)]
    assert len(set(keys)) == 3 and not synced
    assert search(4, 64) == (keys[0], True)                  # used again: the next to go is the one of 128
    fourth, known = search(4, 512)
    assert not known and beam_keys(g) == [keys[2], keys[0], fourth] and len(synced) == 1
    assert not search(4, 128)[1] and beam_keys(g) == [keys[0], fourth, keys[1]]
    for n in range(64, 4096, 64):
        search(8, n)
        assert len(beam_keys(g)) <= 3
    runner.ctx.workspace.generation = 2                      # scratch has moved: none of them can be replayed
    search(2, 100)
    assert len(beam_keys(g)) == 1 and g._recorded[4, True, False] is decode


@pytest.mark.gpu
def test_searches_of_many_lengths(tmp_path, monkeypatch):
    """Recordings come and go between searches and decoding requests; results are those of an engine that has recorded nothing else."""
    from inferloop_b200 import Engine
    folder, vocab = make_model_folder(str(tmp_path / "m"), *CONFIGS["D"][:2]), CONFIGS["D"][0]["vocab_size"]
    make = lambda: Engine(folder, dtype="float32", block_size=16, num_gpu_blocks_override=400, max_num_seqs=16)  # noqa: E731
    prompts = {n: random_tokens(n, vocab, n) for n in (10, 90, 200, 400)}
    alone = {n: make().beam_search([p], 3, 6, eos_tokens=[])[0] for n, p in prompts.items()}
    monkeypatch.setattr(graphs, "BEAM_STEPS_KEPT", 2, raising=False)
    engine = make()
    greedy = engine.generate([prompts[10]], max_new_tokens=6)
    decoding = set(engine.runner.graphs._recorded)
    for n in (10, 90, 200, 10, 400, 90, 90, 10):
        found = engine.beam_search([prompts[n]], 3, 6, eos_tokens=[])[0]
        assert [(h.tokens, h.score) for h in found] == [(h.tokens, h.score) for h in alone[n]]
        assert len(beam_keys(engine.runner.graphs)) <= 2
    assert engine.generate([prompts[10]], max_new_tokens=6) == greedy and decoding <= set(engine.runner.graphs._recorded)
