"""Beam search's host side without a device: what it refuses, which pages it asks for and how it lays them out."""
from types import SimpleNamespace

import pytest
import torch

from fake_runner import FakeRunner
from inferloop_b200.cache import CacheManager, OutOfPages
from inferloop_b200.engine.beams import BeamSearch
from inferloop_b200.parts.base import CacheNeeds, PagedKVNeed


def search(needs, page, pages, slots, beams, last, stops=()):
    cache = CacheManager(needs, page, pages, slots)
    runner = SimpleNamespace(cache=cache, spec=SimpleNamespace(token_extras=(), vocab_size=100), graphs=SimpleNamespace(whole=True), device=torch.device("cpu"))
    return BeamSearch(SimpleNamespace(runner=runner), beams, last, stops), cache


def test_refusals():
    from inferloop_b200 import Engine
    engine = Engine({}, runner=FakeRunner())
    with pytest.raises(ValueError, match="recorded as one graph"):
        engine.beam_search([[1, 2]], 2, 4)
    with pytest.raises(ValueError, match="vocabulary"):
        engine.beam_search([[50]], 2, 4)
    with pytest.raises(ValueError, match="limit"):
        engine.beam_search([[1] * 510], 2, 4)
    needs = [CacheNeeds(paged=PagedKVNeed(1, 16, None))]
    for beams, last, stops in ((0, 4, ()), (33, 4, ()), (2, 0, ()), (32, 4, (1, 2))):
        with pytest.raises(ValueError):
            search(needs, 4, 16, 4, beams, last, stops)


def test_tensors_off_the_device_are_refused():
    from inferloop_b200.csrc import ops
    f, i = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.beam_select(torch.zeros(8, 10), f, i, i, f)
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.BeamState([([torch.zeros(2, 3, 1, 16, 8)], 16, 1)], [], "cpu")
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.step_build(i, i, i, i, i, i, [], i)
    with pytest.raises(ops.KernelError, match="CUDA only"):
        ops.attention_beams(f, f, f, f, SimpleNamespace(positions=i), i, 2, 0, 1.0, 1, 1, 4)


@pytest.mark.parametrize("prompt,last", [(1, 1), (4, 1), (5, 1), (7, 6), (8, 9), (13, 30), (16, 17)])
@pytest.mark.parametrize("needs", [[PagedKVNeed(1, 16)], [PagedKVNeed(1, 16), PagedKVNeed(2, 16, 6)], [PagedKVNeed(1, 16, 8), PagedKVNeed(1, 16, None, None, 4)]])
@pytest.mark.parametrize("beams", [1, 3])
def test_pages_are_laid_out_for_the_whole_search(prompt, last, needs, beams):
    """Full pages of the prompt in every row, a last page of each row's own, and exactly the pages behind it in the free list that steps of one token a
    row will take, no page twice."""
    page, n_req = 4, 2
    s, cache = search([CacheNeeds(paged=n) for n in needs], page, 200, 8, beams, last)
    prompts = [[1] * prompt, [1] * (prompt + 3)]
    assert s.batch_of(prompts) == 2
    ids = [(s, r, w) for r in range(n_req) for w in range(beams)]
    slots = []
    for r, p in enumerate(prompts):
        slots.append(cache.begin(ids[r * beams]))
        cache.ensure(ids[r * beams], len(p))
        cache.commit(ids[r * beams], len(p))
        for w in range(1, beams):
            slots.append(cache.begin(ids[r * beams + w]))
            cache.ensure(ids[r * beams + w], s._beam_tokens(len(p), len(p) + last - 1))
        cache.ensure(ids[r * beams], len(p) + last - 1)
    bucket, n = n_req * beams + 1, n_req * beams
    i32 = lambda *shape: torch.full(shape, 99, dtype=torch.int32)  # noqa: E731
    ctx = SimpleNamespace(n_seqs=bucket, tokens=i32(bucket), positions=i32(bucket), kv_len=i32(bucket), slots=i32(bucket), seq_of_token=i32(bucket),
                          cu_q=i32(bucket + 1), logit_rows=i32(bucket), block_tables={g.index: i32(bucket, 40) for g in cache.groups})
    pages, ones = s._layout(prompts, ids, slots, ctx)
    assert ones.tolist() == [1] * n and ctx.slots.tolist() == slots + [-1] and ctx.kv_len.tolist()[:n] == [len(p) for p in prompts for _ in range(beams)]
    for g, pg in zip(cache.groups, pages):
        table, free = ctx.block_tables[g.index].tolist(), pg.free.tolist()
        used = [x for row in table for x in row if x >= 0]
        assert not set(used) & set(free) and len(set(free)) == len(free) and all(x == -1 for x in table[n])
        need = 0
        for r, p in enumerate(prompts):
            have, total = len(p) // g.need.stride, (len(p) + last - 1) // g.need.stride
            full, part = have // page, have % page != 0
            rows = table[r * beams:(r + 1) * beams]
            first = cache.block_table(g.index, ids[r * beams])
            assert all(row[:full] == first[:full] for row in rows)
            if part:
                assert len({row[full] for row in rows}) == beams and rows[0][full] == first[full] >= 0
            assert all(x == -1 for row in rows for x in row[full + part:])
            need += beams * (-(-total // page) - full - part)
        assert len(free) == need
    for i in ids:
        cache.release(i)
    cache.check()


def test_batches_follow_slots_and_pages():
    needs = [CacheNeeds(paged=PagedKVNeed(1, 16))]
    s, _ = search(needs, 4, 1000, 10, 3, 5)
    assert s.batch_of([[1] * 9] * 8) == 3                       # ten slots
    s, _ = search(needs, 4, 1000, 2000, 3, 5)
    assert s.batch_of([[1] * 9] * 200) == 85                    # 256 rows of a step
    s, cache = search(needs, 4, 20, 30, 3, 5)                   # 9 + 4 tokens: four pages, the others' two each
    assert s._pages(9) == {0: 4 + 2 * 2} and s.batch_of([[1] * 9] * 5) == 2
    cache.begin("x")
    cache.ensure("x", 60)
    with pytest.raises(OutOfPages):
        s.batch_of([[1] * 9])
    s, cache = search(needs, 4, 20, 2, 3, 5)
    with pytest.raises(OutOfPages, match="slots"):
        s.batch_of([[1]])
