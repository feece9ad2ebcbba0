"""Beam search by its definition: every hypothesis anew through a function from tokens to the logits behind them, lists of lists, 64 bits."""
import math

import numpy as np


def search(logits_of, prompt, beams, last, stops, penalty, early):
    """logits_of([token lists]) -> rows.  Returns ([(tokens, score)] best first, smallest gap between two scores down to the first that is not used)."""
    live, done, over, gap = [([], 0.0)], [], False, math.inf
    for step in range(last):
        rows = logits_of([prompt + t for t, _ in live])
        cands = []
        for b, ((toks, score), x) in enumerate(zip(live, rows)):
            x = np.asarray(x, dtype=np.float64)
            lp = x - (x.max() + math.log(np.exp(x - x.max()).sum()))
            cands += [(score + float(v), float(x[i]), b, i) for i, v in enumerate(lp)]
        k = beams * (1 + len(stops))
        cands.sort(key=lambda c: (-c[0], -c[1], c[2], c[3]))
        nxt, ends, last_used = [], [], k - 1
        for rank, (s, _, b, tok) in enumerate(cands[:k]):
            toks = live[b][0] + [tok]
            if tok in stops:
                if rank < beams:
                    ends.append((toks, s))
            elif len(nxt) < beams:
                nxt.append((toks, s))
                last_used = rank
                if step + 1 == last:
                    ends.append((toks, s))
        for a, b in zip(cands[:last_used + 1], cands[1:last_used + 2]):
            gap = min(gap, a[0] - b[0])
        length = float(step + 1) ** penalty
        for toks, s in ends:
            if len(done) == beams and not s / length > done[-1][1]:
                continue
            done.append((toks, s / length))
            done.sort(key=lambda d: -d[1])
            del done[beams:]
        if not nxt or step + 1 == last or (len(done) == beams and (early or not cands[0][0] / length > done[-1][1])):
            break
        live = nxt
    return done, gap
