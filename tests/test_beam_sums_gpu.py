"""The sums of exponentials that order a selection's beams, to the bound that the kernel's choice between 32 and 64 bits rests on."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("V", [1, 65, 2049, 32003, 151936, 1 << 20])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["normal", "flat", "falling", "one high", "far"])
def test_scores(V, dtype, kind):
    """With p = exp(-d) / sum the share of a logit d below the row's largest: a term's exponent, d log2(e), is off by (2^-23 + 2^-26) d relative to the term, the
    three exponentials on its way by 2^-22 each, sums of 32 bits (64 logits by 11 roundings, ten segments by 11 more) by 22 * 2^-24; what follows is of 64 bits.
    The logarithm of the sum is off by the mean of that, and the mean of d is ln V at most.  The score is rounded once more."""
    from inferloop_b200.csrc import ops
    gen = torch.Generator().manual_seed(V)
    x = {"normal": lambda: 3 * torch.randn(3, V, generator=gen), "flat": lambda: torch.full((3, V), 0.7) + 1e-3 * torch.randn(3, V, generator=gen),
         "falling": lambda: -torch.rand(3, V, generator=gen).mul(1 / V).add(1e-9).log().neg().mul(1.0),
         "one high": lambda: torch.randn(3, V, generator=gen).index_fill(1, torch.tensor([V // 2]), 9.0),
         "far": lambda: 40 * torch.randn(3, V, generator=gen) + 1000.0}[kind]().to(dtype)
    scores = torch.tensor([[-0.25], [-17.0], [-700.0]])
    parents, tokens = (torch.zeros(3, 4, dtype=torch.int32, device=DEV) for _ in range(2))
    out = torch.zeros(3, 4, device=DEV)
    ops.beam_select(x.to(DEV), scores.to(DEV), parents, tokens, out)
    for r, row in enumerate(x.double().numpy()):
        top = row.max()
        lse = top + math.log(np.exp(row - top).sum())
        bound = (2 ** -23 + 2 ** -26) * math.log(V) + 3 * 2 ** -22 + 22 * 2 ** -24
        for token, score in zip(tokens[r].tolist(), out[r].tolist()):
            if token < 0:
                assert V < 4 and score == -math.inf
                continue
            want = float(scores[r, 0]) + float(row[token]) - lse
            assert abs(score - want) <= bound + 2 ** -24 * abs(want) * (1 + 1e-6) + 1e-12 * (1 + abs(top))
