"""What an engine's beams have in the cache, followed through a search bit by bit: after every reordering a beam has what its parent had before it, in every
page group (windows, pooled rows, 4-bit pages) and in every state slot."""
import importlib

import pytest
import torch

from helpers import CONFIGS, make_model_folder, random_tokens
from test_beam_engine_gpu import engine_for

pytestmark = pytest.mark.gpu


def held(cache, tables, slots, lens):
    """Per row: the bytes of all that its tokens have in pages, group by group, and of its slot; None for an entry whose page is not held."""
    rows = []
    for i, n in enumerate(lens):
        parts = []
        for g, table in zip(cache.groups, tables):
            have = n // g.need.stride
            ids = table[i, :-(-have // g.page_size)].tolist()
            for x in (g.storage, g.storage_v):
                if x is None:
                    continue
                unit = g.page_size // x.shape[-2]
                for b, page in enumerate(ids):
                    filled = min(have - b * g.page_size, g.page_size)
                    parts.append(None if page < 0 else x[..., page, :, :-(-filled // unit), :].contiguous().view(torch.uint8).clone())
        for x in cache._slot_state.values():
            parts.append(x[int(slots[i])].clone().flatten().view(torch.uint8))
        rows.append(parts)
    return rows


@pytest.fixture
def followed(monkeypatch):
    """Every reordering of a search is looked at; the number of rows that took a parent's place or were copied."""
    from inferloop_b200.csrc import ops
    plain, seen = ops.beam_reorder, dict(rows=0, calls=0, moved=0)

    def reorder(state, parents, kv_len, tables, slots=None):
        cache = seen["cache"]
        lens = kv_len.tolist()
        before = held(cache, tables, slots, lens)
        plain(state, parents, kv_len, tables, slots)
        after = held(cache, tables, slots, lens)
        W = parents.shape[1]
        for r, line in enumerate(parents.tolist()):
            for w, p in enumerate(line):
                if p < 0:
                    continue
                for a, b in zip(after[r * W + w], before[r * W + p]):
                    assert (a is None) == (b is None) and (a is None or torch.equal(a, b)), (seen["calls"], r, w, p)
                seen["rows"] += 1
                seen["moved"] += p != w
        # the last, partly filled pages and the slots are still a row's own
        for g, table in zip(cache.groups, tables):
            for r in range(len(parents)):
                have = lens[r * W] // g.need.stride
                if have % g.page_size:
                    last = table[r * W:(r + 1) * W, have // g.page_size].tolist()
                    assert len(set(last)) == W and min(last) >= 0
        assert slots is None or len(set(slots.tolist())) == slots.numel()
        seen["calls"] += 1
    monkeypatch.setattr(ops, "beam_reorder", reorder)
    return seen


def follow(engine, seen, vocab, beams, last):
    seen["cache"] = engine.runner.cache
    found = engine.beam_search([random_tokens(n, vocab, 900 + n) for n in (5, 38)], beams, last, 0.0, eos_tokens=[])
    assert seen["calls"] == last - 1 and seen["rows"] == 2 * beams * (last - 1) and seen["moved"] > 0
    assert all(len(x) == beams and all(len(h.tokens) == last for h in x) for x in found)


@pytest.mark.parametrize("name,dtype,kw", [("A", "float32", {}), ("E", "float32", {}), ("D", "bfloat16", {}), ("F", "bfloat16", {}),
                                           ("D", "bfloat16", dict(kv_cache="int4")), ("E", "bfloat16", dict(kv_cache="int4")), ("D", "float32", dict(kv_cache="int4"))])
def test_pages(tmp_path, followed, name, dtype, kw):
    config, seed, page = CONFIGS[name][:3]
    engine = engine_for(make_model_folder(str(tmp_path / "m"), config, seed), dtype, 16 if kw else page, **kw)
    follow(engine, followed, config["vocab_size"], 4, 20)


@pytest.mark.parametrize("family", ["mamevik", "zebivik", "sapanex", "tamovik", "dalavik", "sufolix"])
def test_pages_and_states(tmp_path, followed, family):
    cases = importlib.import_module(family + "_cases")
    for name in sorted(cases.CASES):
        engine = engine_for(cases.folder(str(tmp_path), name, torch.float32), page=cases.CASES[name][2], pages=300, seqs=16)
        if engine.runner.graphs is not None and engine.runner.graphs.whole and not engine.runner.spec.token_extras:
            follow(engine, followed, engine.runner.spec.vocab_size, 3, 18)
            return
    pytest.skip("no configuration of the family is one recorded step")
