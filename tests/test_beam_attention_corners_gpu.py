"""Attention of beams where a launch's CTAs have nothing to do and where values lie at the type's ends, against the plain form in 64 bits."""
import pytest
import torch

from test_beam_attention_gpu import BF, F32, case, check, ops, queries  # noqa: F401 (ops: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_queries_that_are_no_numbers_beside_ctas_without_keys(ops, dtype, d, odd):  # noqa: F811
    """The split follows the longest request, so that most CTAs of a short one have no key: what one beam's queries hold reaches no other beam's
    rows, and a beam that sees nothing gets zeros."""
    nq, nkv, W = 8, 2, 4
    k, v, table, positions = case(3, W, [3000, 20, 1], nkv, d, 16, d, dtype=dtype)
    positions[6] = -1
    q = queries(3 * W, nq, d, dtype, 4)
    for row in (5, 9):
        q[row] = odd
    for _ in range(20):
        out = check(ops, q, k, v, table, positions, W, 0, d ** -0.5, nq, nkv)
        assert (out[6] == 0).all()
