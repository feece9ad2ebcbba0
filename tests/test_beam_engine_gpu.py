"""Beam search through the engine against beam search by its definition, whose logits come from whole prompts run anew.

In 32 bits the engine's logits x at a position do not depend on how the tokens were cut into steps beyond 1e-5 (1 + |x|), the bound of every engine
test: a token's log probability is off by twice that, and two hypotheses of n tokens are in order for sure when their scores differ
by 4 n 1e-5 (1 + max |x|).  Prompts are the first of their seeds whose reference keeps all that it ranks so far apart.
"""
import pytest
import torch

import beam_reference
from helpers import CONFIGS, make_model_folder, random_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("beam_models")
    return {n: make_model_folder(str(root / n), CONFIGS[n][0], CONFIGS[n][1]) for n in CONFIGS}


def engine_for(folder, dtype="float32", page=16, pages=400, seqs=48, **kw):
    from inferloop_b200 import Engine
    return Engine(folder, dtype=dtype, block_size=page, num_gpu_blocks_override=pages, max_num_seqs=seqs, **kw)


def from_whole_prompts(engine):
    """Logits behind token lists, each list a prompt of its own, released afterwards."""
    from inferloop_b200.engine import StepEntry
    r, serial = engine.runner, [0]

    def logits_of(lists):
        out = []
        for toks in lists:
            serial[0] += 1
            name = ("reference", serial[0])
            out.append(r.step([StepEntry(name, toks, [len(toks) - 1])])[0].double().cpu().numpy())
            r.end(name)
        return out
    return logits_of


def decided(engine, lengths, beams, last, stops=(), penalty=1.0, early=False, seed=0, stops_behind=()):
    """[(prompt, stop tokens, reference, bound of a score)] of the given lengths.  stops_behind: stop tokens are those of these ranks behind the prompt."""
    vocab, logits_of, out = engine.runner.spec.vocab_size, from_whole_prompts(engine), []
    for n in lengths:
        for turn in range(200):
            prompt = random_tokens(n, vocab, 1000 * seed + 37 * n + turn)
            ends = set(stops)
            if stops_behind:
                best = (-logits_of([prompt])[0]).argsort()
                ends = {int(best[i]) for i in stops_behind}
            most = [0.0]

            def watched(lists):
                rows = logits_of(lists)
                most[0] = max(most[0], max(float(abs(x).max()) for x in rows))
                return rows
            ref, gap = beam_reference.search(watched, prompt, beams, last, ends, penalty, early)
            bound = 2 * last * 1e-5 * (1 + most[0])
            if gap > 2 * bound:
                out.append((prompt, sorted(ends), ref, bound))
                break
        else:
            raise AssertionError("no prompt keeps its scores apart")
    return out


def compare(engine, lengths, beams, last, penalty=1.0, early=False, **kw):
    cases = decided(engine, lengths, beams, last, penalty=penalty, early=early, **kw)
    if all(c[1] == cases[0][1] for c in cases):
        found = engine.beam_search([c[0] for c in cases], beams, last, penalty, early, cases[0][1])
    else:
        found = [engine.beam_search([c[0]], beams, last, penalty, early, c[1])[0] for c in cases]
    free = engine.runner.cache.free_pages()
    assert not engine.runner.cache.live_requests() and all(free[g.index] == g.pool.num_pages for g in engine.runner.cache.groups)
    engine.runner.cache.check()
    for (_, stops, ref, bound), hyps in zip(cases, found):
        assert [h.tokens for h in hyps] == [t for t, _ in ref]
        for h, (toks, score) in zip(hyps, ref):
            assert abs(h.score - score) <= bound * max(1.0, len(toks) ** -penalty) + 2.0 ** -21 * abs(score)
            assert h.finish_reason == ("eos" if toks[-1] in stops else "length")


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E", "F"])
def test_prompts_of_several_lengths(folders, name):
    """Groups of pages with windows, pages of 4, 8 and 16 tokens, prompts that end inside a page and on its border."""
    page = CONFIGS[name][2]
    engine = engine_for(folders[name], page=page)
    compare(engine, (1, page, 2 * page + 3, 3 * page - 1), 4, page + 2)


@pytest.mark.parametrize("beams,last,stops,penalty,early", [(1, 12, (), 1.0, False), (2, 1, (), 1.0, False), (5, 7, (3, 17), 0.0, False), (6, 8, (5,), 1.0, True),
                                                            (3, 7, (1, 2, 3, 4), 2.0, False), (12, 4, (), -0.5, False)])
def test_beams_stops_and_penalties(folders, beams, last, stops, penalty, early):
    engine = engine_for(folders["D"])
    compare(engine, (9, 30), beams, last, penalty, early, stops_behind=stops)


def test_one_beam_is_greedy(folders):
    engine = engine_for(folders["D"])
    prompt = random_tokens(21, CONFIGS["D"][0]["vocab_size"], 3)
    assert engine.beam_search([prompt], 1, 12, eos_tokens=[])[0][0].tokens == engine.generate([prompt], max_new_tokens=12)[0]


def test_more_prompts_than_run_at_once(folders):
    """Batches of prompts as slots and pages allow, beside requests that are being served."""
    vocab = CONFIGS["D"][0]["vocab_size"]
    engine = engine_for(folders["D"], pages=60, seqs=14)
    other = engine.submit(random_tokens(20, vocab, 77), max_new_tokens=12)
    for _ in range(3):
        engine.step()
    prompts = [random_tokens(5 + 3 * i, vocab, 100 + i) for i in range(9)]
    found = engine.beam_search(prompts, 4, 8, eos_tokens=[])
    while not engine.is_idle():
        engine.step()
    alone = engine_for(folders["D"])
    assert engine.result(other).generated == alone.generate([random_tokens(20, vocab, 77)], max_new_tokens=12)[0]
    for p, hyps in zip(prompts, found):
        one = alone.beam_search([p], 4, 8, eos_tokens=[])[0]
        assert [h.tokens for h in hyps] == [h.tokens for h in one]


def test_what_does_not_fit(folders):
    from inferloop_b200.cache import OutOfPages
    vocab = CONFIGS["D"][0]["vocab_size"]
    engine = engine_for(folders["D"], pages=12, seqs=8)
    with pytest.raises(OutOfPages):
        engine.beam_search([random_tokens(100, vocab, 1)], 4, 40)
    with pytest.raises(OutOfPages):
        engine.beam_search([random_tokens(10, vocab, 1)], 9, 4)
    engine.runner.cache.check()
    assert not engine.runner.cache.live_requests()
    for kw in (dict(beams=0), dict(beams=33), dict(max_new_tokens=0), dict(beams=32, eos_tokens=[1, 2]), dict(length_penalty=float("nan")),
               dict(max_new_tokens=5000)):
        with pytest.raises(ValueError):
            engine.beam_search([[1, 2, 3]], **{**dict(beams=2, max_new_tokens=4), **kw})
    for prompts in ([[]], [[vocab]], [[-1]]):
        with pytest.raises(ValueError):
            engine.beam_search(prompts, 2, 4)
    assert engine.beam_search([], 2, 4) == []


@pytest.mark.parametrize("name,kw", [("D", {}), ("F", {}), ("E", {}), ("D", dict(kv_cache="int4")), ("E", dict(kv_cache="int4"))])
def test_bfloat16_scores(folders, name, kw):
    """In bfloat16 two ways to the same logits differ by its rounding: a hypothesis's score is that of its tokens, run through the same engine as
    one prompt, to the engine tests' bfloat16 bound a token (4 bits: their tests' bound on top); the same search gives the same result twice."""
    vocab = CONFIGS[name][0]["vocab_size"]
    engine = engine_for(folders[name], dtype="bfloat16", **kw)
    prompts = [random_tokens(n, vocab, 60 + n) for n in (17, 40)]
    found = engine.beam_search(prompts, 4, 24, 0.0, eos_tokens=[])
    assert [[h.tokens for h in x] for x in engine.beam_search(prompts, 4, 24, 0.0, eos_tokens=[])] == [[h.tokens for h in x] for x in found]
    from inferloop_b200.engine import StepEntry
    for p, hyps in zip(prompts, found):
        assert [h.score for h in hyps] == sorted((h.score for h in hyps), reverse=True) and len({tuple(h.tokens) for h in hyps}) == 4
        for h in hyps:
            toks = p + h.tokens[:-1]
            rows = engine.runner.step([StepEntry("again", toks, list(range(len(p) - 1, len(toks))))]).double().cpu()
            engine.runner.end("again")
            lp = torch.log_softmax(rows, 1)[torch.arange(len(h.tokens)), torch.tensor(h.tokens)]
            bound = len(h.tokens) * 2 * (1e-2 + (5e-2 if kw else 0.0)) * float(rows.abs().max())
            assert abs(float(lp.sum()) - h.score) <= bound


CASES = [("mamevik", "V"), ("mamevik", "W"), ("mamevik", "Z"), ("zebivik", None), ("sapanex", None), ("tamovik", None), ("dalavik", None), ("sufolix", None)]


@pytest.mark.parametrize("family,case", CASES)
def test_states_follow_the_beams(tmp_path_factory, family, case):
    """Recurrent states, convolutions, previous tokens, latents, pooled blocks and looped layers: every family of models, its first configuration that the
    recorded step takes (Mamevik: three)."""
    import importlib
    cases = importlib.import_module(family + "_cases")
    root = str(tmp_path_factory.mktemp("beam_" + family))
    tried = 0
    for name in ([case] if case else sorted(cases.CASES)):
        config, _, page = cases.CASES[name][:3]
        engine = engine_for(cases.folder(root, name, torch.float32), page=page, pages=200, seqs=16)
        if engine.runner.graphs is None or not engine.runner.graphs.whole or engine.runner.spec.token_extras:
            continue
        tried += 1
        compare(engine, (3, 26), 3, 10)
        if tried == 2:
            break
    if tried == 0:
        with pytest.raises(ValueError, match="recorded as one graph"):
            engine.beam_search([[1, 2]], 2, 2)


@pytest.mark.parametrize("tc_rows", [1, 10 ** 9])
@pytest.mark.parametrize("name", ["D", "F", "E"])
def test_bfloat16_scores_with_shared_pages(folders, monkeypatch, name, tc_rows):
    """The same where pages are read once for all beams however little that is, by either kernel."""
    from inferloop_b200.csrc import ops
    monkeypatch.setattr(ops, "BEAMS_SHARE_BYTES", 0)
    monkeypatch.setattr(ops, "BEAMS_TC_ROWS", tc_rows)
    test_bfloat16_scores(folders, name, {})
    ops.check_device_errors()


def test_a_short_search_leaves_a_long_one_as_it_is(folders):
    vocab = CONFIGS["D"][0]["vocab_size"]
    prompts = [random_tokens(n, vocab, 80 + n) for n in (700, 650)]

    def long(engine):
        return [[(h.tokens, h.score) for h in x] for x in engine.beam_search(prompts, 4, 8, eos_tokens=[])]
    first = long(engine_for(folders["D"], dtype="bfloat16"))
    engine = engine_for(folders["D"], dtype="bfloat16")
    engine.beam_search([p[:20] for p in prompts], 4, 8, eos_tokens=[])
    assert long(engine) == first
