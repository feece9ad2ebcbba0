"""Beam search's selection, reordering and step building on the device against the plain forms."""
import math
import random

import pytest
import torch

import beam_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NEG = float("-inf")


@pytest.fixture(scope="module")
def ops():
    from inferloop_b200.csrc import ops
    return ops


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).to(DEV)


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------------------ selection
def select(ops, logits, scores, k, expect_flags=True):
    R, W = scores.shape
    parents, tokens = (torch.full((R, k), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    out, bad = torch.full((R, k), 77.0, device=DEV), torch.full((R * W,), 77, dtype=torch.int32, device=DEV)
    ops.beam_select(logits.to(DEV) if not logits.is_cuda else logits, scores.to(DEV), parents, tokens, out, bad if expect_flags else None)
    return parents.cpu(), tokens.cpu(), out.cpu(), bad.cpu()


def check_select(ops, logits, scores, k):
    """Beams and tokens exactly; a score within 2 roundings of 32 bits of it and of the sum of exponentials' (each term's argument, up to
    |x - max| <= 100, is rounded by 2^-24 and scaled by a constant that is off by 2^-25, the exponential by 2 steps, and a sum of 2^5 terms a thread and 2^8
    threads by 13 steps): 2^-24 |s| + 2^-23 * (100 * 1.5 + 15) is 2e-5 at most, and far less for the terms that matter."""
    parents, tokens, out, bad = select(ops, logits, scores, k)
    found, flags = plain.select(logits, scores, k)
    assert bad.tolist() == flags
    for r, (p, t, s) in enumerate(found):
        assert parents[r].tolist() == p and tokens[r].tolist() == t, f"request {r}"
        for a, b in zip(out[r].tolist(), s):
            assert a == b if math.isinf(b) else abs(a - b) <= 2e-5 + 2 ** -23 * abs(b)
    return parents, tokens, out


@pytest.mark.parametrize("R,W,V,k", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 6), (1, 4, 8191, 8), (3, 5, 8192, 10), (2, 4, 8193, 8), (1, 2, 32003, 64),
                                     (7, 5, 32003, 15), (2, 32, 3001, 64), (1, 8, 151936, 16), (5, 4, 151936, 8), (64, 4, 40000, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select(ops, R, W, V, k, dtype):
    logits = (3 * randn(R * W, V, seed=V + k)).to(dtype)
    check_select(ops, logits, -30 * torch.rand(R, W, generator=torch.Generator().manual_seed(3)), k)


@pytest.mark.parametrize("V,k", [(300, 64), (20000, 8), (20000, 64)])
def test_select_equal_logits(ops, V, k):
    """Rows of one value, of few values, and the largest values side by side in one thread's reach: the lowest beam, then the lowest token."""
    rows = [torch.zeros(V), torch.full((V,), -3.5), torch.arange(V).remainder(3).float(), torch.arange(V).float() * 1e-3,
            -torch.arange(V).float() * 1e-3, torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)]
    crowd = torch.full((V,), -9.0)
    crowd[128:132] = 5.0
    for j in range(8):
        crowd[(1024 * j + 40) % V:(1024 * j + 44) % V] = 4.0 + j
    rows.append(crowd)
    logits = torch.stack(rows)
    check_select(ops, logits, torch.zeros(1, 7), k)
    check_select(ops, logits, torch.zeros(7, 1), k)
    check_select(ops, torch.stack([rows[2]] * 6), torch.zeros(2, 3), k)                 # whole beams alike


def test_select_masked_and_broken_rows(ops):
    V, k = 9000, 8
    x = randn(12, V, seed=5)
    x[0, 1:] = NEG                      # one token left
    x[1] = NEG                          # none
    x[2, 77] = float("nan")
    x[3, V - 1] = float("inf")
    x[4, :8192] = NEG                   # a whole run of the row
    x[5] = -3.0e38                      # far down, and the type's lowest
    x[6, 5] = torch.finfo(torch.float32).max
    x[7, 4] = torch.finfo(torch.float32).min
    scores = torch.zeros(4, 3)
    check_select(ops, x, scores, k)
    scores[0, 0], scores[2] = NEG, torch.tensor([NEG, NEG, NEG])
    scores[3] = torch.tensor([float("nan"), -1.0, NEG])
    check_select(ops, x, scores, k)
    check_select(ops, x[:3], torch.zeros(1, 3), 5)      # a single candidate in all


def test_select_first_step(ops):
    logits = randn(8, 50000, seed=9)
    scores = torch.full((2, 4), NEG)
    scores[:, 0] = 0
    parents, _, _ = check_select(ops, logits, scores, 8)
    assert (parents == 0).all()


def test_select_strides_and_alignment(ops):
    wide = torch.zeros(6, 10007, device=DEV)
    wide.copy_(randn(6, 10007, seed=2))
    for a, b in ((0, 10007), (1, 9000), (3, 8196), (4, 9001)):
        view = wide[:, a:b]
        got = select(ops, view, torch.zeros(2, 3), 6)
        found, _ = plain.select(view, torch.zeros(2, 3), 6)
        assert [x.tolist() for x in got[:2]] == [[f[0] for f in found], [f[1] for f in found]]
    half = wide.bfloat16()[::2, 5:9005]
    got = select(ops, half, torch.zeros(1, 3), 6, expect_flags=False)
    found, _ = plain.select(half, torch.zeros(1, 3), 6)
    assert got[0][0].tolist() == found[0][0] and got[1][0].tolist() == found[0][1] and (got[3] == 77).all()


def test_select_scores_in_place(ops):
    """The new scores may be written over the old ones, also where the beams come so close that their sums are taken again."""
    near = randn(1, 40000, seed=5)
    rows = torch.cat([near, near.flip(1), 3 * randn(1, 40000, seed=6), near.roll(7, 1)])
    for logits, R in ((rows, 1), (3 * randn(12, 9001, seed=7), 3)):
        scores = -torch.arange(logits.shape[0], dtype=torch.float32).remainder(2).view(R, 4) / 64
        parents, tokens, out, bad = select(ops, logits, scores, 4)
        x, again = scores.to(DEV), [torch.zeros((R, 4), dtype=torch.int32, device=DEV) for _ in range(2)]
        ops.beam_select(logits.to(DEV), x, *again, x)
        assert torch.equal(x.cpu(), out) and torch.equal(again[0].cpu(), parents) and torch.equal(again[1].cpu(), tokens)


@pytest.mark.parametrize("R,W,V,k", [(3, 1, 2048, 64), (1, 3, 700, 64), (40, 2, 33000, 4), (150, 2, 6000, 8), (1, 32, 70000, 64), (9, 6, 50000, 12)])
def test_select_sizes_between(ops, R, W, V, k):
    logits = 3 * randn(R * W, V, seed=V)
    check_select(ops, logits, -5 * torch.rand(R, W, generator=torch.Generator().manual_seed(4)), k)


@pytest.mark.parametrize("R,W,V,k,gap", [(2, 12, 58754, 24, 4.0), (1, 16, 13900, 32, 9.0), (3, 8, 9573, 24, 30.0), (1, 32, 40000, 64, 50.0), (2, 2, 2048, 64, 100.0),
                                         (1, 2, 5000, 64, 100.0), (1, 32, 700, 64, 1.0), (1, 3, 151936, 64, 20.0), (2, 16, 1073, 48, 5.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_scores_far_apart(ops, R, W, V, k, gap, dtype):
    """One or a few beams bring all that is found; with bfloat16 logits, many equal ones."""
    scores = torch.stack([-gap * torch.randperm(W, generator=torch.Generator().manual_seed(r)).float() for r in range(R)])
    check_select(ops, (2 * randn(R * W, V, seed=V + W)).to(dtype), scores, k)


def test_select_two_streams_and_graph(ops):
    """Two selections on two streams at once, and a recorded one beside them, each with scratch of its own."""
    R, W, V, k = 2, 4, 60000, 8
    xs = [randn(R * W, V, seed=s).to(DEV) for s in range(3)]
    scores = torch.zeros(R, W, device=DEV)
    outs = [[torch.zeros(R, k, dtype=torch.int32, device=DEV), torch.zeros(R, k, dtype=torch.int32, device=DEV), torch.zeros(R, k, device=DEV)] for _ in xs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.beam_select(xs[2], scores, *outs[2])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for st, x, o in zip(streams, xs, outs):
            with torch.cuda.stream(st):
                ops.beam_select(x, scores, *o)
        graph.replay()
    torch.cuda.synchronize()
    for x, o in zip(xs, outs):
        found, _ = plain.select(x, scores, k)
        assert o[0].tolist() == [f[0] for f in found] and o[1].tolist() == [f[1] for f in found]
    xs[2].copy_(xs[0])
    graph.replay()
    torch.cuda.synchronize()
    assert outs[2][1].tolist() == outs[0][1].tolist()


# ------------------------------------------------------------------ what goes on and what is finished
@pytest.mark.parametrize("W,n_stops,early,penalty", [(1, 1, False, 1.0), (3, 1, False, 1.0), (4, 2, True, 0.0), (5, 0, False, 1.0), (8, 3, False, 2.0),
                                                     (16, 3, True, -0.5), (32, 1, False, 1.0)])
def test_keep(ops, W, n_stops, early, penalty):
    R, steps, k = 5, 7, min(64, W * (n_stops + 1))
    rng = random.Random(W)
    track = ops.BeamTrack.make(R, W, steps, DEV)
    states = [dict(done=[], over=False) for _ in range(R)]
    stops = list(range(n_stops))
    for step in range(steps):
        cands = []
        for r in range(R):
            n = k if rng.random() < 0.8 else rng.randint(0, k)
            pairs = rng.sample([(w, t) for w in range(W) for t in range(40 if r % 2 else 6)], min(n, 6 * W))
            s = sorted((float(torch.tensor(-rng.random() * 9, dtype=torch.float32)) for _ in pairs), reverse=True)
            cands.append([(w, t, x) for (w, t), x in zip(pairs, s)] + [(-1, -1, NEG)] * (k - len(pairs)))
        ops.beam_keep(i32([[c[0] for c in x] for x in cands]), i32([[c[1] for c in x] for x in cands]),
                      torch.tensor([[c[2] for c in x] for x in cands], device=DEV), i32(stops) if stops else None, track, step, steps, penalty, early)
        for r in range(R):
            live = plain.keep(cands[r], stops, W, step, steps, penalty, early, states[r])
            pad = W - len(live)
            assert track.parents[r].tolist() == [x[0] for x in live] + [-1] * pad == track.past_parents[step, r].tolist()
            assert track.tokens[r].tolist() == [x[1] for x in live] + [0] * pad == track.past_tokens[step, r].tolist()
            assert track.scores[r].tolist() == [x[2] for x in live] + [NEG] * pad
            done = states[r]["done"]
            n = int(track.done_count[r])
            assert n == len(done) and bool(track.done[r]) == states[r]["over"], (step, r)
            for i, (score, at, parent, token) in enumerate(done):
                # (a power and a division in 32 bits: 4 steps)
                assert abs(float(track.done_scores[r, i]) - score) <= 2 ** -21 * abs(score)
                assert [int(x[r, i]) for x in (track.done_steps, track.done_parents, track.done_tokens)] == [at, parent, token]


# ------------------------------------------------------------------ reordering
def reorder_case(seed, R, W, lens, groups, slot_shapes, parents=None):
    """groups: (outer shape, heads, page, row, dtype, stride, unit); returns CPU tensors."""
    gen = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    made = []
    for outer, heads, page, row, dtype, stride, unit in groups:
        have = [n // stride for n in lens]
        blocks = [-(-n // page) for n in have]
        width = max(blocks) + 2
        rows = []
        for r in range(R):
            shared = [("s", r, b) for b in range(blocks[r])]
            for w in range(W):
                line = list(shared)
                for b in range(blocks[r]):
                    if rng.random() < 0.3:
                        line[b] = (r, b, w % 2)
                if blocks[r] and have[r] % page:
                    line[-1] = (r, w, "last")
                rows.append(line)
        ids = {}
        for line in rows:
            for key in line:
                ids.setdefault(key, len(ids))
        pool = len(ids) + 2
        order = torch.randperm(pool, generator=gen)
        table = torch.full((R * W, width), -1, dtype=torch.int32)
        for i, line in enumerate(rows):
            for b, key in enumerate(line):
                table[i, b] = int(order[ids[key]])
        table[:, width - 1] = 99 + torch.arange(R * W)          # an entry behind the rows in use stays
        if dtype == torch.uint8:
            x = torch.randint(0, 256, (*outer, pool, heads, page // unit, row), generator=gen).to(torch.uint8)
        else:
            x = torch.randn(*outer, pool, heads, page, row, generator=gen).to(dtype)
        made.append((table, [x], page, stride, unit))
    slots = torch.randperm(R * W + 3, generator=gen)[:R * W].to(torch.int32)
    states = [torch.randn(R * W + 3, *s, generator=gen).to(dt) if dt.is_floating_point else torch.randint(0, 100, (R * W + 3, *s), generator=gen).to(dt)
              for s, dt in slot_shapes]
    if parents is None:
        parents = torch.tensor([[rng.choice([rng.randrange(W), min(rng.randrange(W), rng.randrange(W)), -1 if rng.random() < 0.1 else 0]) for _ in range(W)]
                                for _ in range(R)], dtype=torch.int32)
    kv_len = torch.tensor([n for n in lens for _ in range(W)], dtype=torch.int32)
    return parents, kv_len, made, slots, states


def run_reorder(ops, parents, kv_len, groups, slots, states, times=1):
    on = lambda t: t.to(DEV)  # noqa: E731
    g = [(on(t), [on(x) for x in xs], page, stride) for t, xs, page, stride, _ in groups]
    s, st = on(slots), [on(x) for x in states]
    state = ops.BeamState([(xs, page, stride) for _, xs, page, stride in g], st, DEV)
    for _ in range(times):
        ops.beam_reorder(state, on(parents), on(kv_len), [t for t, _, _, _ in g], s)
        plain.reorder(parents, kv_len, groups, slots, states)
    for (t, xs, _, _), (t0, xs0, _, _, _) in zip(g, groups):
        assert torch.equal(t.cpu(), t0)
        for x, x0 in zip(xs, xs0):
            assert torch.equal(x.cpu().view(torch.uint8), x0.view(torch.uint8))
    assert torch.equal(s.cpu(), slots)
    for x, x0 in zip(st, states):
        assert torch.equal(x.cpu().view(torch.uint8).flatten() if x.dim() else x.cpu(), x0.view(torch.uint8).flatten() if x0.dim() else x0)


BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


@pytest.mark.parametrize("R,W,lens", [(1, 1, [5]), (1, 2, [16]), (1, 4, [17]), (3, 5, [0, 1, 33]), (2, 8, [31, 200]), (4, 16, [15, 16, 17, 64]), (2, 32, [40, 47]),
                                      (64, 4, [10 + i for i in range(64)])])
def test_reorder(ops, R, W, lens):
    run_reorder(ops, *reorder_case(R + W, R, W, lens, [((3, 2), 2, 16, 64, BF, 1, 1)], [((5, 7), F32)]), times=3)


@pytest.mark.parametrize("groups", [
    [((2, 2), 1, 16, 32, F32, 1, 1)], [((2, 2), 3, 64, 96, BF, 1, 1)], [((4,), 2, 32, 18 * 64, U8, 1, 16)], [((4,), 2, 16, 18 * 32, U8, 1, 16)],
    [((2, 2), 2, 16, 64, BF, 1, 1), ((2, 2), 2, 16, 64, BF, 16, 1)], [((2,), 1, 16, 5, BF, 1, 1)], [((2,), 1, 16, 3, F32, 1, 1), ((1,), 2, 128, 33, F32, 3, 1)],
    []])
def test_reorder_storages(ops, groups):
    """Types, page sizes, packed pages, rows that stand for several tokens, rows of odd size, and no pages at all."""
    run_reorder(ops, *reorder_case(len(groups) + 5, 3, 4, [23, 61, 130], groups, [((), torch.int32), ((1025,), F32), ((3, 341), BF), ((4096,), F32)]), times=2)


def test_reorder_every_child_of_one_and_none(ops):
    for parents in ([[2, 2, 2, 2]], [[0, 1, 2, 3]], [[3, 2, 1, 0]], [[-1, -1, -1, -1]], [[1, -1, 1, 0]], [[0, 0, -1, -1]]):
        run_reorder(ops, *reorder_case(1, 1, 4, [21], [((2, 2), 2, 16, 64, BF, 1, 1)], [((9,), F32)], torch.tensor(parents, dtype=torch.int32)))


def test_reorder_in_a_pool_of_more_than_32_bits(ops):
    pages = (1 << 32) // (8 * 16 * 128 * 2) + 9
    x = torch.empty((1, pages, 8, 16, 128), dtype=BF, device=DEV)
    x[:, -8:] = randn(1, 8, 8, 16, 128, seed=9).to(BF).to(DEV)
    was, table = x[:, -8:].clone(), torch.tensor([[pages - 8 + i] for i in range(8)], dtype=torch.int32, device=DEV)
    state = ops.BeamState([([x], 16, 1)], [], DEV)
    ops.beam_reorder(state, i32([[1, 1, 3, 3], [2, 0, 0, 0]]), i32([11] * 4 + [16 * 1 - 1] * 4), [table], None)
    for row, (source, fill) in enumerate(((1, 11), (1, 11), (3, 11), (3, 11), (6, 15), (4, 15), (4, 15), (4, 15))):
        assert torch.equal(x[0, int(table[row, 0]), :, :fill], was[0, source, :, :fill])
    assert sorted(table.flatten().tolist()) == list(range(pages - 8, pages))


def test_reorder_pages_that_are_not_held(ops):
    """A window let the first pages go; a row whose last page is missing, or outside the pool, moves nothing there."""
    parents, kv_len, groups, slots, states = reorder_case(4, 2, 4, [70, 71], [((2, 2), 2, 16, 64, BF, 1, 1)], [((9,), F32)])
    table = groups[0][0]
    table[:, :2] = -1
    table[5, 4] = -1
    table[2, 4] = 100000
    run_reorder(ops, parents, kv_len, groups, slots, states)


# ------------------------------------------------------------------ steps laid out on the device
def run_build(ops, new, cached, geometry, extra_tokens=0, in_place=False, spare=3, width_more=2):
    """geometry: [(page, stride)]."""
    S, total = len(new), sum(new)
    groups, pages = [], []
    gen = torch.Generator().manual_seed(S)
    for page, stride in geometry:
        had = [-(-(c // stride) // page) for c in cached]
        need = sum(-(-((c + n) // stride) // page) - h for n, c, h in zip(new, cached, had))
        width = max([-(-((c + n) // stride) // page) for n, c in zip(new, cached)] + [1]) + width_more
        pool = torch.randperm(sum(had) + need + spare, generator=gen).to(torch.int32)
        table = torch.full((S, width), -1, dtype=torch.int32)
        used = 0
        for s, h in enumerate(had):
            table[s, :h] = pool[used:used + h]
            used += h
        if had and had[0] > 1:
            table[0, 0] = -1                    # let go by a window
        groups.append([table.tolist(), pool.tolist(), used, page, stride])
        pages.append(ops.StepPages(table.to(DEV), pool.to(DEV), i32([used]), page, stride))
    full = lambda n, dt=torch.int32: torch.full((n,), -7, dtype=dt, device=DEV)  # noqa: E731
    positions, seq, cu, slot_map, refused = full(total + extra_tokens), full(total + extra_tokens), full(S + 1), full(total + extra_tokens, torch.int64), i32([0])
    before = i32(cached)
    kv_len = before if in_place else full(S)
    ops.step_build(i32(new), before, kv_len, positions, seq, cu, pages, refused, slot_map=slot_map if geometry and geometry[0][1] == 1 else None)
    assert int(refused) == 0
    cu0, len0, pos0, seq0, map0 = plain.build(new, cached, groups)
    assert cu.tolist() == cu0 and kv_len.tolist() == len0
    assert positions.tolist() == pos0 + [-7] * extra_tokens and seq.tolist() == seq0 + [-7] * extra_tokens
    if geometry and geometry[0][1] == 1:
        assert slot_map.tolist() == map0 + [-7] * extra_tokens
    for g, p in zip(groups, pages):
        assert p.table.tolist() == g[0] and int(p.used) == g[2]


@pytest.mark.parametrize("new,cached,geometry", [
    ([1], [0], [(16, 1)]), ([1], [15], [(16, 1)]), ([1], [16], [(16, 1)]), ([0], [3], [(16, 1)]), ([0, 0], [0, 0], [(16, 1)]),
    ([5, 0, 1, 40, 0], [16, 7, 31, 0, 0], [(16, 1)]), ([1] * 33, list(range(33)), [(16, 1), (16, 16)]), ([3, 2000, 1], [5, 100, 4000], [(64, 1), (16, 4), (32, 1)]),
    ([7, 1], [2, 2], []), ([2048] * 5, [0] * 5, [(128, 1)]), ([1] * 257, [i % 19 for i in range(257)], [(1, 1)]), ([9, 9], [3, 3], [(16, 3)]),
    ([1, 0, 2, 1], [4, 4, 4, 4], [(16, 1)]), ([0, 0, 3], [15, 16, 17], [(16, 1), (24, 5)])])
def test_build(ops, new, cached, geometry):
    run_build(ops, new, cached, geometry)
    run_build(ops, new, cached, geometry, extra_tokens=5, in_place=True, spare=0, width_more=0)


def test_build_many_sequences(ops):
    rng = random.Random(1)
    run_build(ops, [rng.choice([0, 1, 1, 1, 13]) for _ in range(8192)], [rng.randrange(100) for _ in range(8192)], [(16, 1)], in_place=True)


@pytest.mark.parametrize("change,bit", [("tokens", 1), ("pages", 2), ("columns", 4), ("negative", 8), ("negative cached", 8), ("too long", 8), ("used", 2)])
def test_build_refuses_whole_steps(ops, change, bit):
    """Nothing is written but the bit."""
    new, cached = [4, 20, 1], [3, 5, 16]
    table, free, used = torch.full((3, 4), -1, dtype=torch.int32, device=DEV), i32(list(range(9))), i32([2])
    room = 25
    if change == "tokens":
        room = 24
    elif change == "pages":
        free = free[:3]                         # two pages are needed and two are taken
    elif change == "columns":
        table = table[:, :1].contiguous()
    elif change == "negative":
        new[1] = -1
    elif change == "negative cached":
        cached[2] = -5
    elif change == "too long":
        cached[0] = 2 ** 31 - 2
    else:
        used = i32([-1])
    full = lambda n: torch.full((n,), -7, dtype=torch.int32, device=DEV)  # noqa: E731
    kv, pos, seq, cu, refused = full(3), full(room), full(room), full(4), i32([0])
    slot_map = torch.full((room,), -7, dtype=torch.int64, device=DEV)
    t0, u0 = table.clone(), int(used)
    ops.step_build(i32(new), i32(cached), kv, pos, seq, cu, [ops.StepPages(table, free, used, 16)], refused, slot_map=slot_map)
    assert int(refused) & bit and all((x == -7).all() for x in (kv, pos, seq, cu, slot_map)) and torch.equal(table, t0) and int(used) == u0


# ------------------------------------------------------------------ refusals
def test_refusals(ops):
    z = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    f = torch.float32
    x, sc, p, o = z(8, 100, dt=f), z(2, 4, dt=f), z(2, 8), z(2, 8, dt=f)
    for args in ((x[:7], sc, p, p, o), (x, sc, p, z(2, 7), o), (x, sc, z(2, 65), z(2, 65), z(2, 65, dt=f)), (x, sc.double(), p, p, o), (x, sc, p.long(), p, o),
                 (x.half(), sc, p, p, o), (x.t().contiguous().t(), sc, p, p, o), (z(8, 0, dt=f), sc, p, p, o), (x[:1].expand(8, 100), sc, p, p, o),
                 (z(66, 100, dt=f), z(2, 33, dt=f), p, p, o), (x, sc, p, p, o, z(7))):
        with pytest.raises(ops.KernelError):
            ops.beam_select(*args)
    ops.beam_select(z(0, 100, dt=f), z(0, 4, dt=f), z(0, 8), z(0, 8), z(0, 8, dt=f))            # no request: nothing to do
    cache, table = z(2, 2, 9, 2, 16, 64, dt=f), z(8, 4)
    state = ops.BeamState([([cache], 16, 1)], [z(8, 5, dt=f)])
    for args in ((state, z(2, 4), z(8), [], z(8)), (state, z(2, 4), z(8), [table[:7].contiguous()], z(8)), (state, z(2, 4), z(7), [table], z(8)),
                 (state, z(2, 4), z(8), [table], None), (state, z(8), z(8), [table], z(8)), (state, z(2, 4, dt=torch.int64), z(8), [table], z(8)),
                 (state, z(2, 33), z(66), [z(66, 4)], z(66)), (state, z(512, 4), z(2048), [z(2048, 4)], z(2048))):
        with pytest.raises(ops.KernelError):
            ops.beam_reorder(*args)
    for groups, slots in (([([cache], 8, 1)], []), ([([cache[0, 0]], 24, 1)], []), ([([], 16, 1)], []), ([([cache, cache[:, :, :5].contiguous()], 16, 1)], []),
                          ([([cache.transpose(0, 2)], 16, 1)], []), ([], [z(8, 5), z(7, 5)]), ([([cache], 16, 0)], []), ([([cache.cpu()], 16, 1)], [])):
        with pytest.raises(ops.KernelError):
            ops.BeamState(groups, slots, DEV)
    a, r = z(3), z(1)
    page = lambda **kw: ops.StepPages(**{**dict(table=z(3, 2), free=z(5), used=z(1), page_size=16), **kw})  # noqa: E731
    for args, kw in (((a, z(2), a, z(4), z(4), z(4), [page()], r), {}), ((a, a, a, z(4), z(3), z(4), [page()], r), {}), ((a, a, a, z(4), z(4), z(3), [page()], r), {}),
                     ((a, a, a, z(4), z(4), z(4), [page(table=z(2, 2))], r), {}), ((a, a, a, z(4), z(4), z(4), [page(page_size=0)], r), {}),
                     ((a, a, a, z(4), z(4), z(4), [page()] * 9, r), {}), ((a, a, a, z(4), z(4), z(4), [page(stride=2)], r), dict(slot_map=z(4, dt=torch.int64))),
                     ((a, a, a, z(4), z(4), z(4), [page()], r), dict(slot_map=z(4))), ((z(9000), z(9000), z(9000), z(4), z(4), z(9001), [], r), {})):
        with pytest.raises(ops.KernelError):
            ops.step_build(*args, **kw)
    track = ops.BeamTrack.make(2, 4, 3, DEV)
    c = (z(2, 8), z(2, 8), z(2, 8, dt=f))
    for args in ((*c, None, track, 3, 3), (*c, None, track, 2, 2), (z(1, 8), *c[1:], None, track, 0, 3), (c[0], c[1], c[1], None, track, 0, 3)):
        with pytest.raises(ops.KernelError):
            ops.beam_keep(*args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [2041, 2048, 2049, 4089, 6144, 1])
def test_select_rows_that_begin_anywhere(ops, dtype, V):
    """Rows at every place of a 16-byte vector, the best tokens at their ends."""
    for offset in range(0, 9, 1 if V == 2041 else 4):
        base = torch.full((6, V + 16), 50.0)                # (what lies beside a row is larger than all of it)
        base[:, offset:offset + V] = 2 * randn(6, V, seed=V + offset)
        for w in range(6):
            base[w, offset] += 4.0 + w / 16
            base[w, offset + V - 1] += 4.5 + w / 32
        x = base.to(dtype).to(DEV)[:, offset:offset + V]
        parents, tokens, out, bad = select(ops, x, torch.zeros(2, 3), 5)
        found, flags = plain.select(x.cpu(), torch.zeros(2, 3), 5)
        for r, (p, t, s) in enumerate(found):
            assert parents[r].tolist() == p and tokens[r].tolist() == t and not bad.any()
            assert all(a == b or abs(a - b) <= 2e-5 + 2 ** -23 * abs(b) for a, b in zip(out[r].tolist(), s))
