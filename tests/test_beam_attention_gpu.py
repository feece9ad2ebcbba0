"""Attention of beams that share pages against the plain form in 64 bits."""
import random
from types import SimpleNamespace

import pytest
import torch

import beam_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(params=["few rows", "tcgen05"])
def ops(request, monkeypatch):
    """Every case through the kernels of few rows, and again with all that the tcgen05 kernel takes sent there."""
    from inferloop_b200.csrc import ops
    monkeypatch.setattr(ops, "BEAMS_TC_ROWS", 1 if request.param == "tcgen05" else 10 ** 9)
    monkeypatch.setattr(ops, "BEAMS_TC_FEW", 10 ** 9)
    yield ops
    ops.check_device_errors()


def case(R, W, lens, nkv, d, page, seed, rows=None, dtype=BF, shared=0.7, spare=2):
    """(k, v, table, positions) on the CPU: rows of request r have lens[r] keys; of each block, beams share a page with odds `shared`."""
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    ids, lines = {}, []
    for r in range(R):
        blocks = -(-lens[r] // page)
        owner = [[0] * W if rng.random() < shared else [rng.randrange(W) for _ in range(W)] for _ in range(blocks)]
        if blocks and lens[r] % page:
            owner[-1] = list(range(W))
        lines += [[(r, b, owner[b][w]) for b in range(blocks)] for w in range(W)]
    for line in lines:
        for key in line:
            ids.setdefault(key, len(ids))
    pool = len(ids) + spare
    order = torch.randperm(pool, generator=gen).tolist()
    table = torch.full((R * W, max([len(x) for x in lines] + [1]) + 2), -1, dtype=torch.int32)
    for i, line in enumerate(lines):
        for b, key in enumerate(line):
            table[i, b] = order[ids[key]]
    positions = torch.tensor([lens[r] - 1 for r in range(R) for _ in range(W)], dtype=torch.int32)
    k, v = (torch.randn(pool, nkv, page, d, generator=gen).to(dtype) for _ in range(2))
    n = R * W if rows is None else rows
    return k, v, table[:n].contiguous(), positions[:n].contiguous()


def make_step(positions, longest=None):
    n = positions.numel()
    step = SimpleNamespace(positions=positions.to(DEV), seq_of_token=torch.arange(n, dtype=torch.int32, device=DEV))
    if longest:
        step.max_kv_len = longest
    return step


def bound(q, out, mass, most, L, d):
    """Of a row and head with scores up to `most` (sums of |q_i k_i| scale): a score is off by d + 4 roundings of 32 bits at most (a truncating
    adder: 2^-23 each), which the softmax's quotient doubles; exponentials by 2^-22, sums over the keys and the records by L + 64 roundings of
    2^-23; with bfloat16 weights rounded once (2^-8), and the output rounded once."""
    most = most.repeat_interleave(d, 1)
    low = q.dtype == BF
    rel = 2 * (d + 4) * 2.0 ** -23 * most + (L + 64) * 2.0 ** -23 + 2.0 ** -21 + (2.0 ** -8 if low else 0.0)
    half = torch.finfo(q.dtype).eps / 2
    return mass * rel * (1 + half) + out.abs() * half + 1e-30


def check(ops, q, k, v, table, positions, W, window, scale, nq, nkv, sink=None, longest=None):
    d = q.shape[1] // nq
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    ops.attention_beams(q.to(DEV), out, k.to(DEV), v.to(DEV), make_step(positions, longest), table.to(DEV), W, window, scale, nq, nkv, d,
                        sink=None if sink is None else sink.to(DEV))
    ref, mass, most = plain.attention(q, k, v, positions, table, window, scale, nq, nkv, sink)
    err = (out.cpu().double() - ref).abs()
    lim = bound(q, ref, mass, most, int(positions.max()) + 1, d)
    assert torch.equal(torch.isnan(err), torch.isnan(ref))
    assert bool((err.nan_to_num(0.0) <= lim.nan_to_num(1.0)).all()), f"{float((err / lim).nan_to_num(0.0).max())} times the bound at row {int((err / lim).nan_to_num(0.0).argmax()) // q.shape[1]}"
    return out.cpu()


def queries(rows, nq, d, dtype, seed):
    return (1.5 * torch.randn(rows, nq * d, generator=torch.Generator().manual_seed(seed + 1000))).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nq,nkv,d", [(4, 4, 32), (8, 2, 64), (6, 2, 96), (8, 2, 128), (5, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize("W,R", [(1, 3), (2, 2), (3, 2), (4, 3), (8, 2), (32, 1)])
def test_attention(ops, dtype, nq, nkv, d, W, R):
    """Every number of rows a CTA has, from one to more than one CTA takes."""
    lens = [70, 1, 33][:R]
    k, v, table, positions = case(R, W, lens, nkv, d, 16, W + d, dtype=dtype)
    check(ops, queries(R * W, nq, d, dtype, 3), k, v, table, positions, W, 0, d ** -0.5, nq, nkv)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window,sink", [(0, False), (40, False), (1, True), (-32, False), (-1, True), (500, True)])
def test_windows_pages_and_sinks(ops, dtype, page, window, sink):
    nq, nkv, d, W = 8, 2, 64, 4
    k, v, table, positions = case(3, W, [129, 300, 64], nkv, d, page, page + window, dtype=dtype, rows=11)      # (the last request has three rows)
    s = torch.randn(nq, generator=torch.Generator().manual_seed(1)) if sink else None
    check(ops, queries(11, nq, d, dtype, 4), k, v, table, positions, W, window, d ** -0.5, nq, nkv, s)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("W,nkv,G,n", [(4, 1, 4, 2500), (16, 1, 2, 1100), (2, 1, 16, 3000), (32, 1, 1, 700)])
def test_many_keys(ops, dtype, W, nkv, G, n):
    """Lists of units that are made in several goes, clusters of many CTAs; and a length that the plan did not know."""
    d = 64
    k, v, table, positions = case(1, W, [n], nkv, d, 16, n, dtype=dtype, shared=0.5)
    q = queries(W, nkv * G, d, dtype, 5)
    a = check(ops, q, k, v, table, positions, W, 0, 0.2, nkv * G, nkv)
    check(ops, q, k, v, table, positions, W, 0, 0.2, nkv * G, nkv, longest=17)
    assert torch.equal(a, check(ops, q, k, v, table, positions, W, 0, 0.2, nkv * G, nkv))          # the same bits each time


@pytest.mark.parametrize("dtype", [BF, F32])
def test_many_requests(ops, dtype):
    """More CTAs than are resident at once."""
    nq, nkv, d, W, R = 8, 2, 128, 4, 90
    lens = [20 + (7 * r) % 50 for r in range(R)]
    k, v, table, positions = case(R, W, lens, nkv, d, 16, 8, dtype=dtype)
    check(ops, queries(R * W, nq, d, dtype, 6), k, v, table, positions, W, 0, d ** -0.5, nq, nkv)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,page", [(64, 32), (128, 16), (96, 64), (48, 16), (64, 8)])
def test_rows_of_their_own_lengths_and_pages_that_are_not_held(ops, dtype, d, page):
    """Rows of one request at different positions, one at -1, one behind its table, pages that are missing or outside the pool; heads and pages
    that the fast kernels are not built for."""
    nq, nkv, W = 4, 2, 4
    k, v, table, positions = case(2, W, [150, 90], nkv, d, page, d, dtype=dtype)
    positions[1], positions[2], positions[5] = 20, -1, 10 ** 6
    table[3, 1], table[0, :] = 10 ** 6, -1
    table[6, 2:] = -7
    for window in (0, 30, -64):
        out = check(ops, queries(8, nq, d, dtype, 7), k, v, table, positions, W, window, d ** -0.5, nq, nkv)
        assert (out[0] == 0).all() and (out[2] == 0).all()
    check(ops, queries(8, nq, d, dtype, 7), k, v, table, positions, W, 0, d ** -0.5, nq, nkv, sink=torch.tensor([0.5, -3.0, float("-inf"), 90.0]))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("W,nq", [(4, 8), (8, 8), (16, 8)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf"), 3e38])
def test_masked_places_hold_anything(ops, dtype, W, nq, what):
    """Keys and values behind a row's length, before its window, and in the pages of other beams do not reach it."""
    nkv, d, n, page = 2, 64, 55, 16
    k, v, table, positions = case(2, W, [n, n], nkv, d, page, 11, dtype=dtype, shared=0.4)
    for i in range(2 * W):
        last = int(table[i, 3])
        k[last, :, n % page:], v[last, :, n % page:] = what, what
    for window in (0, 20):
        check(ops, queries(2 * W, nq, d, dtype, 8), k, v, table, positions, W, window, d ** -0.5, nq, nkv)
    other = int(table[1, 3])                          # (a page of beam 1's own)
    v[other, :, 2] = what
    k[other, 1, 1] = what
    q = queries(2 * W, nq, d, dtype, 8)
    out = torch.zeros(q.shape, dtype=dtype, device=DEV)
    ops.attention_beams(q.to(DEV), out, k.to(DEV), v.to(DEV), make_step(positions), table.to(DEV), W, 0, d ** -0.5, nq, nkv, d)
    ref, mass, most = plain.attention(q, k, v, positions, table, 0, d ** -0.5, nq, nkv)
    rest = [i for i in range(2 * W) if i != 1]
    lim = bound(q, ref, mass, most, n, d)
    assert bool(((out.cpu().double() - ref).abs()[rest] <= lim[rest]).all())
    if what == what and abs(what) > 3.1e38:           # an infinity that is seen: none of the row's head is a plain number
        assert not torch.isfinite(out.cpu()[1, :d]).any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lowest_and_largest_scores(ops, dtype):
    """Scores at the type's ends, and rows of equal ones."""
    nq, nkv, d, W = 4, 1, 32, 2
    k, v, table, positions = case(1, W, [40], nkv, d, 16, 5, dtype=dtype)
    for scale in (0.0, 1e-30, -0.3, 1e4):
        q = queries(W, nq, d, dtype, 9)
        check(ops, q, k, v, table, positions, W, 0, scale, nq, nkv)


def test_streams_and_graphs(ops):
    """A recorded call replayed beside others on another stream; the table that it reads changes in between."""
    nq, nkv, d, W, dtype = 8, 2, 64, 4, BF
    k, v, table, positions = case(2, W, [100, 77], nkv, d, 16, 2)
    q = queries(8, nq, d, dtype, 1)
    dk, dv, dt, dq, step = k.to(DEV), v.to(DEV), table.to(DEV), q.to(DEV), make_step(positions)
    outs = [torch.zeros(8, nq * d, dtype=dtype, device=DEV) for _ in range(2)]
    args = lambda o: (dq, o, dk, dv, step, dt, W, 0, 0.125, nq, nkv, d)  # noqa: E731
    ops.attention_beams(*args(outs[0]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_beams(*args(outs[0]))
    side = torch.cuda.Stream()
    for shift in (0, 1):
        changed = table.roll(shift, 0)
        dt.copy_(changed)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            ops.attention_beams(*args(outs[1]))
        torch.cuda.synchronize()
        ref, mass, most = plain.attention(q, k, v, positions, changed, 0, 0.125, nq, nkv)
        for o in outs:
            assert bool(((o.cpu().double() - ref).abs() <= bound(q, ref, mass, most, 100, d)).all())
    assert torch.equal(*outs)


def test_unaligned_and_empty(ops):
    nq, nkv, d, W = 4, 2, 64, 2
    k, v, table, positions = case(1, W, [30], nkv, d, 16, 2)
    flat = torch.zeros(k.numel() + 1, dtype=BF, device=DEV)
    dk = flat[1:].view(k.shape)
    dk.copy_(k)
    q = queries(W, nq, d, BF, 1)
    out = torch.zeros(W, nq * d, dtype=BF, device=DEV)
    ops.attention_beams(q.to(DEV), out, dk, v.to(DEV), make_step(positions), table.to(DEV), W, 0, 0.125, nq, nkv, d)
    ref, mass, most = plain.attention(q, k, v, positions, table, 0, 0.125, nq, nkv)
    assert bool(((out.cpu().double() - ref).abs() <= bound(q, ref, mass, most, 30, d)).all())
    ops.attention_beams(q[:0].to(DEV), out[:0], dk, v.to(DEV), make_step(positions[:0]), table[:0].to(DEV), W, 0, 0.125, nq, nkv, d)


def test_refusals(ops):
    nq, nkv, d, W = 4, 2, 64, 2
    k, v, table, positions = (x.to(DEV) for x in case(1, W, [30], nkv, d, 16, 2))
    q = queries(W, nq, d, BF, 1).to(DEV)
    out, step = torch.zeros_like(q), make_step(positions)
    good = dict(q=q, out=out, k=k, v=v, step=step, table=table, beams=W, nq=nq, nkv=nkv, d=d, sink=None)
    for change in (dict(q=q[:1]), dict(q=q.float()), dict(out=out.float()), dict(k=k.float()), dict(v=v[:, :1].contiguous()), dict(k=k.transpose(0, 1)),
                   dict(table=table.long()), dict(table=table[:1]), dict(table=table[:, :0].contiguous()), dict(beams=0), dict(beams=33), dict(nq=5), dict(nkv=0),
                   dict(d=32), dict(sink=torch.zeros(3, device=DEV)), dict(sink=torch.zeros(nq)), dict(q=q.cpu()), dict(step=make_step(positions.long())),
                   dict(k=k[:0], v=v[:0])):
        a = {**good, **change}
        with pytest.raises(ops.KernelError):
            ops.attention_beams(a["q"], a["out"], a["k"], a["v"], a["step"], a["table"], a["beams"], 0, 0.125, a["nq"], a["nkv"], a["d"], sink=a["sink"])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_cache_of_more_than_32_bits(ops, dtype):
    """The pages at the end of a pool of more than 2^32 bytes give the bits that they give in a pool of their own."""
    nq, nkv, d, W, page = 16, 8, 128, 4, 16
    k, v, table, positions = case(2, W, [300, 77], nkv, d, page, 11, dtype=dtype)
    own, pool = k.shape[0], (1 << 32) // (nkv * page * d * k.element_size()) + 50
    q, step = queries(2 * W, nq, d, dtype, 7).to(DEV), make_step(positions)
    outs = []
    for moved in (0, pool - own):
        caches = []
        for x in (k, v):
            big = torch.empty((moved + own, *x.shape[1:]), dtype=dtype, device=DEV)
            big[moved:] = x.to(DEV)
            caches.append(big)
        outs.append(torch.zeros_like(q))
        ops.attention_beams(q, outs[-1], *caches, step, torch.where(table < 0, table, table + moved).to(DEV), W, 0, d ** -0.5, nq, nkv, d)
    assert outs[0].abs().sum() > 0 and torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page,shared", [(48, 0.7), (112, 0.5), (128, 0.0), (80, 0.0)])
def test_large_and_odd_pages(ops, dtype, page, shared):
    """Pages of 3, 7, 8 and 5 strips; beams that hold a page each."""
    nq, nkv, d, W = 8, 1, 64, 8
    k, v, table, positions = case(2, W, [301, 47], nkv, d, page, page, dtype=dtype, shared=shared)
    check(ops, queries(2 * W, nq, d, dtype, 9), k, v, table, positions, W, 0, d ** -0.5, nq, nkv)
    check(ops, queries(2 * W, nq, d, dtype, 9), k, v, table, positions, W, 70, d ** -0.5, nq, nkv)
