"""The plain forms that the operators are tested against, put together to a search and compared with beam search by its definition."""
import math

import numpy as np
import pytest
import torch

import beam_plain as plain
import beam_reference


def model(vocab, seed, spread=3.0):
    """Logits behind a token list, from the tokens alone."""
    def logits_of(lists):
        return [np.random.default_rng([seed, *toks]).standard_normal(vocab) * spread for toks in lists]
    return logits_of


def search(logits_of, prompt, beams, last, stops, penalty, early):
    """One request through beam_plain.select and keep, walked back as the engine does."""
    k, state, past = beams * (1 + len(stops)), dict(done=[], over=False), []
    live = [(0, None, 0.0)]
    texts = [[]]
    for step in range(last):
        rows = torch.from_numpy(np.stack(logits_of([prompt + t for t in texts])))
        (parents, tokens, scores), = plain.select(rows, torch.tensor([[s for _, _, s in live]], dtype=torch.float64), k)[0]
        live = plain.keep(list(zip(parents, tokens, scores)), stops, beams, step, last, penalty, early, state)
        texts = [texts[p] + [t] for p, t, _ in live]
        past.append([(p, t) for p, t, _ in live])
        if state["over"]:
            break
    out = []
    for score, step, beam, token in state["done"]:
        toks = [token]
        for s in range(step - 1, -1, -1):
            toks.append(past[s][beam][1])
            beam = past[s][beam][0]
        out.append((toks[::-1], score))
    return out


@pytest.mark.parametrize("beams,vocab,last,n_stops,penalty,early", [(1, 30, 8, 0, 1.0, False), (4, 50, 7, 1, 1.0, False), (3, 20, 12, 3, 0.0, False), (5, 11, 9, 2, 2.0, True),
                                                                    (8, 6, 5, 0, 1.0, False), (6, 40, 10, 4, -0.5, False), (2, 9, 15, 1, 1.0, True)])
def test_the_plain_forms_make_the_search(beams, vocab, last, n_stops, penalty, early):
    stops = list(range(n_stops))
    for seed in range(12):
        logits_of = model(vocab, seed)
        ref, _ = beam_reference.search(logits_of, [seed, 3], beams, last, set(stops), penalty, early)
        found = search(logits_of, [seed, 3], beams, last, stops, penalty, early)
        assert [t for t, _ in found] == [t for t, _ in ref]
        assert all(math.isclose(a, b, rel_tol=1e-12) for (_, a), (_, b) in zip(found, ref))
