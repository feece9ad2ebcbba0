"""Attention over the 4-bit cache where its number formats are at their ends, held to the bound that kv4_bounds.py derives element by element."""
import pytest
import torch

import kv4_bounds
import kv4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from inferloop_b200.csrc import ops
    return ops


@pytest.fixture
def unpacked(ops, monkeypatch):
    """Every sequence above KV4_SHORT_ROWS has its keys and values unpacked, however little fills the device."""
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", 0)
    calls, inner = [], ops._kv4_portions
    monkeypatch.setattr(ops, "_kv4_portions", lambda *args: (calls.append(1), inner(*args)))
    return calls


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def filled(k, v, page, seed):
    """(cache on the GPU, block table) of one sequence whose keys and values are k, v [L, nkv, d]."""
    L, nkv, d = k.shape
    table, pool = plain.make_table([L], page, 2, seed)
    cache = torch.zeros(pool, nkv, page // 16, 18 * d, dtype=torch.uint8)
    at = torch.arange(L)
    plain.write(cache, table[0, at // page], at % page, k, v)
    return cache.to(DEV), table.to(DEV)


def check(ops, q, cache, table, start, tokens, nq, nkv, window=0, sink=None, unpacked=False, scale=None):
    d = q.shape[1] // nq
    scale = d ** -0.5 if scale is None else scale
    out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device=DEV)
    step = plain.make_step([start], [tokens], DEV)
    ops.kv4_attention(q.to(DEV), out, cache, step, table, window, scale, nq, nkv, d, sink=None if sink is None else sink.to(DEV))
    ref, bound = kv4_bounds.outcome(q, cache, table, [start], [tokens], window, scale, nq, nkv, sink, unpacked)
    err = (out.cpu().double() - ref).abs()
    over = err / bound.clamp(min=1e-300)
    assert bool((err <= bound).all()), f"{float(over.max())} times the bound at {int(over.argmax())}, {float(torch.isnan(err).float().mean())} of it NaN"
    return out


@pytest.mark.parametrize("tokens", [1, 3, 90])
@pytest.mark.parametrize("query,key", [(0.0, 1e-4), (0.0, 1.0), (2.0 ** -120, 2.0 ** -20), (2.0 ** -126, 2.0 ** -100)])
def test_queries_of_nothing_and_next_to_nothing(ops, unpacked, tokens, query, key):
    """Rows of zeros, and rows so small that their scores are: the mean of the values, with masked keys beside."""
    nq, nkv, d, L = 8, 2, 64, 300
    k, v = (randn(L, nkv, d, seed=s).bfloat16() for s in (1, 2))
    cache, table = filled((key * k.double()).bfloat16(), v, 16, 3)
    q = randn(tokens, nq * d, seed=4).double() * query
    q[:, d:2 * d] = 0.0
    check(ops, q.bfloat16(), cache, table, L - tokens, tokens, nq, nkv, unpacked=tokens == 90)
    assert bool(unpacked) == (tokens == 90)
