"""Attention over the 4-bit cache from bfloat16 queries, held element by element to what the number formats may cost (kv4_bounds.py): channels of
every size, so that none hides behind the largest; short and long contexts, whole and cut, by the codes and unpacked."""
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


def inputs(kv, lens, nq, nkv, d, page, seed, sharp=1.5):
    """(queries, cache, block table): values whose channels differ by some powers of e, keys less so."""
    gen = torch.Generator().manual_seed(seed)
    table, pool = plain.make_table(kv, page, 2, seed)
    cache = torch.zeros(pool, nkv, page // 16, 18 * d, dtype=torch.uint8)
    size = torch.exp(torch.randn(2, nkv, d, generator=gen) * torch.tensor([0.3, 1.5])[:, None, None])
    for s, n in enumerate(kv):
        if n:
            at = torch.arange(n)
            k, v = ((torch.randn(n, nkv, d, generator=gen) * x).bfloat16() for x in size)
            plain.write(cache, table[s, at // page], at % page, k, v)
    return (sharp * torch.randn(sum(lens), nq * d, generator=gen)).bfloat16(), cache, table


def case(ops, kv, lens, nq, nkv, d, page=16, window=0, sink=False, seed=1, unpacked=False, sharp=1.5):
    q, cache, table = inputs(kv, lens, nq, nkv, d, page, seed, sharp)
    sinks = torch.randn(nq, generator=torch.Generator().manual_seed(seed)) if sink else None
    starts, scale = [n - k for n, k in zip(kv, lens)], d ** -0.5
    ref, bound = kv4_bounds.outcome(q, cache, table, starts, lens, window, scale, nq, nkv, sinks, unpacked)
    assert float(bound.median()) < 0.2 * float(ref.abs().median())       # (an output of zeros would not pass)
    if ops is None:
        return
    out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device=DEV)
    ops.kv4_attention(q.to(DEV), out, cache.to(DEV), plain.make_step(starts, lens, DEV), table.to(DEV), window, scale, nq, nkv, d,
                      sink=None if sinks is None else sinks.to(DEV))
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= bound).all()), f"{float((err / bound.clamp(min=1e-300)).max())} times the bound at {int((err / bound.clamp(min=1e-300)).argmax())}"


HEADS = [(8, 2, 64), (4, 4, 128), (32, 8, 128), (5, 1, 96), (6, 2, 32), (16, 2, 128), (34, 2, 128), (8, 2, 256), (6, 2, 160)]


@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("window,sink", [(0, False), (100, True), (-64, False)])
def test_single_tokens(ops, nq, nkv, d, window, sink):
    case(ops, [1, 15, 16, 17, 131, 300], [1] * 6, nq, nkv, d, 16, window, sink)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("kv,window", [([5000], 0), ([2500, 2400, 30], 0), ([9000, 8900], 0), ([9000, 50], 4100)])
def test_many_keys(ops, kv, window, page):
    case(ops, kv, [1] * len(kv), 4, 2, 64, page, window, True, sharp=4.5)      # (some keys stand out: what all of them sum to says less the more they are)


@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (32, 8, 128), (5, 1, 96), (8, 2, 256)])
@pytest.mark.parametrize("window", [0, 20, -24])
def test_portions_beside_single_tokens(ops, nq, nkv, d, window):
    case(ops, [61, 19, 36, 77, 101], [1, 19, 3, 70, 1], nq, nkv, d, 16, window, window == 20)


@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (32, 8, 128), (34, 2, 128), (2, 2, 128)])
@pytest.mark.parametrize("window", [0, 40, -100])
def test_unpacked_portions(ops, monkeypatch, nq, nkv, d, window):
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", 0)
    case(ops, [500, 77], [160, 70], nq, nkv, d, 16, window, window == 40, unpacked=True)
    case(ops, [300, 140], [130, 140], nq, nkv, d, 128, window, False, 2, unpacked=True)


def test_long_sequences_among_many_short_ones(ops):
    kv = [1 + 37 * s % 90 for s in range(150)]
    kv[0], kv[75], kv[149] = 5000, 3100, 2500
    case(ops, kv, [1] * 150, 8, 4, 32, 32)
