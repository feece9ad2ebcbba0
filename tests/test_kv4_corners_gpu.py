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


@pytest.mark.parametrize("tokens", [1, 3, 90])
def test_next_to_nothing_against_nearly_everything(ops, unpacked, tokens):
    """Queries of 2^-110 over keys of 2^90 tell nothing apart either."""
    nq, nkv, d, L = 8, 2, 64, 300
    k, v = (randn(L, nkv, d, seed=s).bfloat16() for s in (1, 2))
    cache, table = filled((2.0 ** 90 * k.double()).bfloat16(), v, 16, 3)
    q = (randn(tokens, nq * d, seed=4).double() * 2.0 ** -110).bfloat16()
    check(ops, q, cache, table, L - tokens, tokens, nq, nkv, unpacked=tokens == 90)


def leading(lead, tokens, nq, nkv, d, L, ahead, seed):
    """Queries of one direction with a little noise, and keys of which those in `ahead` stand `lead` before the others in every token's logits."""
    base = randn(nkv, d, seed=seed).double()
    q = (base.repeat_interleave(nq // nkv, 0) + 0.1 * randn(tokens, nq, d, seed=seed + 1).double()).flatten(1).bfloat16()
    k = 0.3 * randn(L, nkv, d, seed=seed + 2).double()
    k[ahead] += base / (base * base).sum(1, keepdim=True) * lead * d ** 0.5
    return q, k.bfloat16()


@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("first,last", [(0, 128), (0, 130), (128, 256), (256, 400), (399, 400), (0, 400)])
@pytest.mark.parametrize("lead,size", [(0, 1e-3), (6, 1.0), (10, 0.02), (8, 1e-30), (5, 1e6)])
def test_tiles_of_values_of_nothing(ops, unpacked, tokens, first, last, lead, size):
    """A tile of 128 keys whose values are all zero weighs what its scores say and takes no precision from the others."""
    nq, nkv, d, L = 8, 2, 64, 400
    ahead = torch.arange(first, last)
    q, k = leading(lead, tokens, nq, nkv, d, L, ahead, 5)
    v = (size * randn(L, nkv, d, seed=9).double()).bfloat16()
    v[ahead] = 0.0
    cache, table = filled(k, v, 16, 3)
    out = check(ops, q, cache, table, L - tokens, tokens, nq, nkv, unpacked=tokens == 90)
    assert bool(unpacked) == (tokens == 90) and (last - first < L or not bool(out.any()))


@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -100, 2.0 ** 60])
def test_long_beginnings_without_values(ops, unpacked, tokens, size):
    """Many tiles of zeros before the first values, which the sum of the weights has to hold; a head with a sink beside."""
    nq, nkv, d, L = 4, 1, 128, 3000
    q, k = leading(4, tokens, nq, nkv, d, L, torch.arange(0, 2700), 15)
    v = (size * randn(L, nkv, d, seed=19).double()).bfloat16()
    v[:2700] = 0.0
    cache, table = filled(k, v, 32, 3)
    check(ops, q, cache, table, L - tokens, tokens, nq, nkv, unpacked=tokens == 90)
    check(ops, q, cache, table, L - tokens, tokens, nq, nkv, sink=randn(nq, seed=1), unpacked=tokens == 90)


@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("lead", [8, 12, 14, 16, 17])
def test_a_first_key_that_only_takes_weight(ops, unpacked, tokens, lead):
    """One key with nearly all the weight and next to no value: what comes out is the others', a 2^-24 of the weights each."""
    nq, nkv, d, L = 8, 2, 64, 700
    q, k = leading(lead, tokens, nq, nkv, d, L, torch.arange(1), 25)
    v = randn(L, nkv, d, seed=29)
    v[0] *= 1e-7
    cache, table = filled(k, v.bfloat16(), 16, 3)
    check(ops, q, cache, table, L - tokens, tokens, nq, nkv, unpacked=tokens == 90)
    assert bool(unpacked) == (tokens == 90)
