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


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("W,nq,d", [(4, 8, 64), (2, 2, 128), (16, 8, 64)])
@pytest.mark.parametrize("n", [2, 55, 3000])
@pytest.mark.parametrize("rising,sink", [(False, False), (True, False), (False, True)])
def test_largest_values_that_are_seen(ops, dtype, W, nq, d, n, rising, sink):  # noqa: F811
    """A mean of finite values is finite: values of 3e38 at all keys or at every third, scores in no order or each a little above the one before.  (The
    bound is that of `check`: it is relative to the mean of the absolute values.)"""
    nkv = 2
    k, v, table, positions = case(2, W, [n, n], nkv, d, 16, n, dtype=dtype)
    q = queries(2 * W, nq, d, dtype, 6)
    if rising:
        q[:] = 0.25
        for i in range(2 * W):
            for at in range(n):
                k[int(table[i, at // 16]), :, at % 16] = 4.0 * at / n
    sign = torch.where(torch.arange(d) % 2 == 0, 1.0, -1.0)
    v[:] = (3e38 * sign).to(dtype)
    s = torch.linspace(-1.0, 3.0, nq) if sink else None
    check(ops, q, k, v, table, positions, W, 0, d ** -0.5, nq, nkv, s)
    v[:, :, ::3] = torch.randn(v[:, :, ::3].shape, generator=torch.Generator().manual_seed(n)).to(dtype)
    check(ops, q, k, v, table, positions, W, 0, d ** -0.5, nq, nkv, s)
