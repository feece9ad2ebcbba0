"""The 4-bit key/value cache's kernels against the plain statement in 64 bits (kv4_plain.py).

Tolerances.  bfloat16 rows are kept exactly as the definition says (a quotient of bfloat16 numbers is a half or far from one), 32-bit
rows but for quotients within a rounding of a half or of a scale's (a share of 1e-4 may be a step off).  What is read back is one
rounding of code times scale.  Attention from 32-bit queries: 2^-20 of the largest value for each unit of the largest score, of which
20 are taken at least (a 32-bit sum of some hundred terms is off by some 2^-22 of its terms, which moves a probability by as much);
from bfloat16 queries: 2^-8 (|ref| + largest value), probabilities and the
result being rounded to bfloat16 once each."""
import pytest
import torch

import kv4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from inferloop_b200.csrc import ops
    return ops


def random_rows(n, nkv, d, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, nkv, d, generator=gen) * torch.exp(torch.randn(nkv, d, generator=gen))).to(dtype)


def filled(kv, nkv, d, page, dtype, seed, spare=2):
    """(cache on the GPU, table) with rows of every sequence written by the plain statement."""
    table, pool = plain.make_table(kv, page, spare, seed)
    cache = torch.zeros(plain_shape(pool, nkv, page, d), dtype=torch.uint8)
    for s, n in enumerate(kv):
        at = torch.arange(n)
        k, v = random_rows(n, nkv, d, dtype, seed + 7 * s), random_rows(n, nkv, d, dtype, seed + 7 * s + 3)
        plain.write(cache, table[s, at // page], at % page, k, v)
    return cache.to(DEV), table.to(DEV)


def plain_shape(pool, nkv, page, d):
    return pool, nkv, page // 16, 18 * d


def read_all(ops, cache, table, kv, dtype):
    pages, nkv, units, width = cache.shape
    out = [torch.full((table.numel(), nkv, units * 16, width // 18), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    to = torch.arange(table.numel(), dtype=torch.int32, device=DEV).view(table.shape)
    ops.kv4_read(cache, table, torch.tensor(kv, dtype=torch.int32, device=DEV), to, *out)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv,d,page", [(2, 32, 16), (1, 64, 32), (3, 96, 16), (8, 128, 16), (2, 128, 128), (2, 256, 64), (1, 512, 16)])
def test_rows_are_kept_as_the_definition_says(ops, dtype, nkv, d, page):
    starts, lens = [0, 5, 40], [17, 1, 33]
    kv = [a + n for a, n in zip(starts, lens)]
    table, pool = plain.make_table(kv, page, 2, 1)
    step = plain.make_step(starts, lens, DEV)
    # views of a projection's rows, and values whose heads come before their tokens
    qkv = random_rows(sum(lens), 2 * nkv + 1, d, dtype, 2)
    k, v = qkv[:, 1:1 + nkv], qkv[:, 1 + nkv:].transpose(0, 1).contiguous().transpose(0, 1)
    cache = torch.randint(0, 256, plain_shape(pool, nkv, page, d), dtype=torch.uint8, generator=torch.Generator().manual_seed(3))
    want = cache.clone()
    pos, seq = step.positions.cpu().long(), step.seq_of_token.cpu().long()
    plain.write(want, table[seq, pos // page], pos % page, k, v)
    got = cache.to(DEV)
    ops.kv4_write(qkv.to(DEV)[:, 1:1 + nkv], v.transpose(0, 1).contiguous().to(DEV).transpose(0, 1), step, table.to(DEV), got)
    got = got.cpu()
    if dtype == torch.bfloat16:
        assert torch.equal(got, want)
    else:
        assert float((got != want).float().mean()) <= 1e-4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 128, 160])
@pytest.mark.parametrize("starts,lens", [([0], [301]), ([7, 0, 250], [130, 1, 175])])
def test_many_rows_are_kept_as_the_definition_says(ops, dtype, d, starts, lens):
    """Steps long enough for the form that takes tokens by fours, cut anywhere, with a page that is not held."""
    nkv, page, T = 3, 32, sum(lens)
    table, pool = plain.make_table([a + n for a, n in zip(starts, lens)], page, 2, 1)
    table[0, 1] = -1
    step = plain.make_step(starts, lens, DEV)
    k, v = random_rows(T, nkv, d, dtype, 11), random_rows(T, nkv, d, dtype, 12)
    want = torch.zeros(plain_shape(pool, nkv, page, d), dtype=torch.uint8)
    pos, seq = step.positions.cpu().long(), step.seq_of_token.cpu().long()
    pages = table[seq, pos // page]
    held = pages >= 0
    plain.write(want, pages[held], (pos % page)[held], k[held], v[held])
    got = torch.zeros_like(want, device=DEV)
    ops.kv4_write(k.to(DEV), v.to(DEV), step, table.to(DEV), got)
    wrong = float((got.cpu() != want).float().mean())
    assert wrong == 0 if dtype == torch.bfloat16 else wrong <= 1e-4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [96, 128])
def test_rows_of_a_long_step_off_their_boundaries(ops, dtype, d):
    starts, lens, nkv, page = [3, 0, 900], [701, 1, 445], 2, 64
    T = sum(lens)
    table, pool = plain.make_table([a + n for a, n in zip(starts, lens)], page, 2, 1)
    table[2, 15] = -1
    step = plain.make_step(starts, lens, DEV)
    x = random_rows(T, 2 * nkv, d + 1, dtype, 13)
    k, v = x[:, :nkv, 1:], x[:, nkv:, 1:]
    want = torch.zeros(plain_shape(pool, nkv, page, d), dtype=torch.uint8)
    pos, seq = step.positions.cpu().long(), step.seq_of_token.cpu().long()
    pages = table[seq, pos // page]
    held = pages >= 0
    plain.write(want, pages[held], (pos % page)[held], k[held], v[held])
    got, x = torch.zeros_like(want, device=DEV), x.to(DEV)
    ops.kv4_write(x[:, :nkv, 1:], x[:, nkv:, 1:], step, table.to(DEV), got)
    wrong = float((got.cpu() != want).float().mean())
    assert wrong == 0 if dtype == torch.bfloat16 else wrong <= 1e-4


@pytest.mark.parametrize("odd", [1, 2, 3])
def test_rows_on_any_element_boundary(ops, odd):
    """Rows that start where no vector load may."""
    step, table = plain.make_step([3], [5], DEV), torch.tensor([[1]], dtype=torch.int32, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        x = random_rows(5, 1, 2 * 64 + 2 * odd, dtype, 4).to(DEV)
        k, v = x[:, :, odd:odd + 64], x[:, :, odd + 64:odd + 128]
        a, b = (torch.zeros(2, 1, 1, 18 * 64, dtype=torch.uint8, device=DEV) for _ in range(2))
        ops.kv4_write(k, v, step, table, a)
        ops.kv4_write(k.contiguous(), v.contiguous(), step, table, b)
        assert torch.equal(a, b) and int(a.sum()) > 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_halves_zeros_and_what_is_not_finite(ops, dtype):
    d, T = 64, 8
    x = torch.zeros(T, 1, d)
    x[0, 0, :32] = torch.arange(-16, 16) * 0.5 * 7 / 8                  # amax 7: s = 1, halves and quarters
    x[1, 0, :8] = torch.tensor([7.0, 0.5, -0.5, 1.5, -1.5, 2.5, 6.5, -6.5])
    x[2, 0, 3], x[2, 0, 40] = float("inf"), 2.0
    x[3, 0, 33], x[3, 0, 0] = float("nan"), -3.0
    x[4, 0, 5] = 2.0 ** -130                                             # a scale below the smallest normal number
    x[5, 0, :32] = 3e38
    x[6, 0, 31] = -float("inf")
    x[7] = -0.0
    x = x.to(dtype)
    step, table = plain.make_step([0], [T], DEV), torch.tensor([[0]], dtype=torch.int32, device=DEV)
    cache = torch.zeros(1, 1, 1, 18 * d, dtype=torch.uint8, device=DEV)
    ops.kv4_write(x.to(DEV), x.flip(0).contiguous().to(DEV), step, table, cache)
    k, v = read_all(ops, cache, table, [T], torch.float32)
    want = plain.kept(x)[2][:, 0]
    assert torch.equal(torch.nan_to_num(k[0, 0, :T].cpu().double(), 99.0), torch.nan_to_num(want, 99.0))
    assert torch.equal(torch.nan_to_num(v[0, 0, :T].cpu().double(), 99.0), torch.nan_to_num(want.flip(0), 99.0))
    assert torch.isnan(k[0, 0, 2, :32]).all() and float(k[0, 0, 2, 40]) != 0 and torch.isnan(k[0, 0, 3, 32:]).all()
    assert k[0, 0, 1, :8].tolist() == [7.0, 1.0, -1.0, 2.0, -2.0, 3.0, 7.0, -7.0]


def test_tokens_without_a_page_are_left_out(ops):
    step = plain.make_step([14, 0, 40], [4, 1, 1], DEV)
    table = torch.tensor([[2, -1], [9, 9], [0, 1]], dtype=torch.int32, device=DEV)      # 9: past the pool; position 40: past the table
    cache = torch.zeros(3, 2, 1, 18 * 32, dtype=torch.uint8, device=DEV)
    x = random_rows(6, 2, 32, torch.bfloat16, 5).to(DEV)
    ops.kv4_write(x, x, step, table, cache)
    want = torch.zeros(3, 2, 1, 18 * 32, dtype=torch.uint8)
    plain.write(want, [2, 2], [14, 15], x[:2].cpu(), x[:2].cpu())
    assert torch.equal(cache.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv,d,page", [(1, 32, 16), (8, 128, 16), (2, 96, 32), (3, 64, 128), (2, 256, 16)])
def test_pages_read_back(ops, dtype, nkv, d, page):
    kv = [0, 1, page, 2 * page + 5, 33]
    cache, table = filled(kv, nkv, d, page, torch.bfloat16, 6)
    table[3, 1] = -1                                                     # a page that went
    k, v = read_all(ops, cache, table, kv, dtype)
    for s, n in enumerate(kv):
        for b in range(table.shape[1]):
            got = [x[s * table.shape[1] + b].cpu() for x in (k, v)]
            live = min(page, n - b * page)
            if live <= 0:
                assert all(bool((x == 7.0).all()) for x in got)          # left alone
                continue
            want = plain.rows(cache, [max(0, int(table[s, b]))])
            for x, w in zip(got, want):
                w = w[0].to(dtype) * (0 if int(table[s, b]) < 0 else 1)
                assert torch.equal(x[:, :live], w[:, :live]) and not bool(x[:, live:].any())


HEADS = [(8, 2, 64), (4, 4, 128), (32, 8, 128), (5, 1, 96), (6, 2, 32), (16, 2, 128), (12, 1, 64), (34, 2, 128), (8, 2, 256), (3, 1, 512)]


def check(ops, dtype, nq, nkv, d, page, starts, lens, window, sink, seed, scale=None, spoil=None):
    kv = [a + n for a, n in zip(starts, lens)]
    cache, table = filled(kv, nkv, d, page, torch.bfloat16, seed)
    if spoil is not None:
        spoil(cache, table)
    gen = torch.Generator().manual_seed(seed + 1)
    q = (1.5 * torch.randn(sum(lens), nq * d, generator=gen)).to(dtype)
    sinks = torch.randn(nq, generator=gen) if sink else None
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((sum(lens), nq * d), 5.0, dtype=dtype, device=DEV)
    step = plain.make_step(starts, lens, DEV)
    ops.kv4_attention(q.to(DEV), out, cache, step, table, window, scale, nq, nkv, d, sink=None if sinks is None else sinks.to(DEV))
    want, most = plain.attention(q, cache, table, starts, lens, window, scale, nq, nkv, sinks)
    top = max(float(torch.nan_to_num(x).abs().max()) for x in plain.rows(cache, list(range(cache.shape[0]))))
    bound = 2.0 ** -20 * max(20.0, most) * top if dtype == torch.float32 else 2.0 ** -8 * (want.abs() + top)
    err = (out.cpu().double() - want).abs()
    assert bool((err <= bound).all()), f"{float(err.max())} at {int(err.argmax())}, largest value {top}"
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", HEADS)
def test_single_tokens(ops, dtype, nq, nkv, d):
    check(ops, dtype, nq, nkv, d, 16, [0, 14, 15, 16, 130, 299], [1] * 6, 0, False, 10)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [32, 64, 128])
@pytest.mark.parametrize("window,sink", [(0, True), (40, False), (1, True), (-32, False), (500, True)])
def test_windows_sinks_and_pages(ops, dtype, page, window, sink):
    check(ops, dtype, 8, 2, 64, page, [0, 31, 39, 41, 200, 63], [1] * 6, window, sink, 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (32, 8, 128), (5, 1, 96), (34, 2, 128), (8, 2, 256)])
@pytest.mark.parametrize("window", [0, 20, -24])
def test_portions_beside_single_tokens(ops, dtype, nq, nkv, d, window):
    check(ops, dtype, nq, nkv, d, 16, [60, 0, 33, 7, 100], [1, 19, 3, 70, 1], window, window == 20, 30)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sequences_that_bring_nothing_and_pages_that_went(ops, dtype):
    def spoil(cache, table):
        table[1, 1] = -1
        table[3] = -1                                                    # a token that sees no key
    out = check(ops, dtype, 8, 2, 64, 16, [5, 50, 0, 20, 3], [0, 2, 0, 1, 1], 0, False, 40, spoil=spoil)
    assert not bool(out[2].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[1, 1, 1], [3, 1, 40]])
def test_what_no_token_sees_may_be_anything(ops, dtype, lens):
    """NaN scales in rows behind the last position, before the window and in pages of nobody."""
    starts, window, nkv, d, page = [40, 77, 5], 30, 2, 64, 32
    nan = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=DEV).repeat(d // 32)
    inf = torch.tensor([0x80, 0x7F], dtype=torch.uint8, device=DEV).repeat(d // 32)

    def spoil(cache, table):
        used = set(table.flatten().tolist())
        for s, (a, n) in enumerate(zip(starts, lens)):
            for key in range(table.shape[1] * page):
                if plain.first_key(a, window) <= key < a + n or int(table[s, key // page]) < 0:
                    continue
                unit = cache[int(table[s, key // page]), :, key % page // 16]
                for base, what in ((16 * d, nan), (17 * d, inf if key % 2 else nan)):
                    at = base + key % 16 * (d // 16)
                    unit[:, at:at + d // 16] = what
        for p in range(cache.shape[0]):
            if p not in used:
                cache[p] = 0xFF
    out = check(ops, dtype, 8, nkv, d, page, starts, lens, window, False, 50, spoil=spoil)
    assert bool(torch.isfinite(out).all())


def test_a_kept_nan_is_seen(ops):
    """A group that holds no number makes the heads that read it NaN, and no others."""
    cache, table = filled([20, 20], 2, 64, 16, torch.bfloat16, 60)
    cache[int(table[0, 0]), 1, 0, 17 * 64 + 3 * 4:17 * 64 + 3 * 4 + 2] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8, device=DEV)
    step = plain.make_step([19, 19], [1, 1], DEV)
    q = torch.randn(2, 4 * 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    out = torch.zeros_like(q)
    ops.kv4_attention(q, out, cache, step, table, 0, 0.125, 4, 2, 64)
    out = out.view(2, 4, 64)
    assert bool(torch.isnan(out[0, 2:, :32]).all()) and not bool(torch.isnan(out[0, 2:, 32:]).any())
    assert not bool(torch.isnan(out[0, :2]).any()) and not bool(torch.isnan(out[1]).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0])
def test_scales_of_scores(ops, dtype, scale):
    """No weight at all, a negative one, and scores so large that one key takes everything."""
    check(ops, dtype, 8, 2, 64, 16, [33, 90], [1, 2], 0, False, 70, scale=scale)


@pytest.mark.parametrize("lens", [[1, 1], [5, 1]])
def test_a_far_key_that_stands_out(ops, lens):
    """One key of many gets nearly all the weight, wherever it lies: what the others added must be scaled down."""
    nq, nkv, d, page, n = 4, 1, 128, 16, 700
    for far in (0, 15, 300, 698):
        cache, table = filled([n, n], nkv, d, page, torch.bfloat16, 80)
        q = torch.randn(sum(lens), nq * d, generator=torch.Generator().manual_seed(2)).bfloat16()
        rows = (20 * q[0, :d].float()).bfloat16().view(1, 1, d)
        host = cache.cpu()
        plain.write(host, [int(table[0, far // page])], [far % page], rows, rows)
        cache = host.to(DEV)
        starts = [n - k for k in lens]
        out = torch.zeros(sum(lens), nq * d, dtype=torch.bfloat16, device=DEV)
        ops.kv4_attention(q.to(DEV), out, cache, plain.make_step(starts, lens, DEV), table, 0, d ** -0.5, nq, nkv, d)
        want, _ = plain.attention(q, cache, table, starts, lens, 0, d ** -0.5, nq, nkv)
        top = max(float(x.abs().max()) for x in plain.rows(cache, list(range(cache.shape[0]))))
        assert bool(((out.cpu().double() - want).abs() <= 2.0 ** -8 * (want.abs() + top)).all())


@pytest.fixture
def unpacked(ops, monkeypatch):
    """Every sequence above KV4_SHORT_ROWS has its keys and values unpacked, however little fills the device."""
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", 0)
    calls, inner = [], ops._kv4_portions
    monkeypatch.setattr(ops, "_kv4_portions", lambda *args: (calls.append(args[5:7]), inner(*args)))
    return calls


@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (32, 8, 128), (34, 2, 128), (2, 2, 128)])
@pytest.mark.parametrize("window", [0, 20, -24])
def test_unpacked_portions_beside_single_tokens(ops, unpacked, nq, nkv, d, window):
    check(ops, torch.bfloat16, nq, nkv, d, 16, [60, 0, 33, 7, 100], [1, 19, 3, 170, 1], window, window == 20, 30)
    assert unpacked


@pytest.mark.parametrize("lens", [[3, 1, 40], [50, 33, 1]])
def test_unpacked_what_no_token_sees_may_be_anything(ops, unpacked, lens):
    test_what_no_token_sees_may_be_anything(ops, torch.bfloat16, lens)
    assert unpacked


@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0])
def test_unpacked_scales_of_scores(ops, unpacked, scale):
    check(ops, torch.bfloat16, 8, 2, 64, 16, [33, 90], [1, 140], 0, False, 70, scale=scale)
    assert bool(unpacked) == (scale > 0)


def test_an_unpacked_far_key_that_stands_out(ops, unpacked):
    test_a_far_key_that_stands_out(ops, [40, 1])
    assert unpacked


@pytest.mark.parametrize("d", [64, 96])
@pytest.mark.parametrize("blocks,tokens", [(1 << 16, 1 << 17), (20, 1 << 17), (1 << 16, 640), (40, 400), (1 << 16, 100)])
def test_runs_of_long_portions(ops, unpacked, monkeypatch, d, blocks, tokens):
    """Long portions beside short ones in groups by what a launch and the scratch take, one too long for the scratch among them."""
    monkeypatch.setattr(ops, "KV4_BLOCKS", blocks)
    monkeypatch.setattr(ops, "KV4_UNPACK_TOKENS", tokens)
    starts, lens = [9, 250, 0, 7, 77, 0, 300, 5], [1, 60, 41, 3, 0, 130, 90, 2]
    check(ops, torch.bfloat16, 8, 2, d, 16, starts, lens, 0, True, 120)
    covered = [s for a, b in unpacked for s in range(a, b)]
    assert covered == ([s for s in (1, 2, 5, 6) if starts[s] + lens[s] <= tokens] if d == 64 else [])


def test_a_portion_on_either_side_of_the_rule(ops, monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "_kv4_portions", lambda *args: calls.append(args[5:7]))
    sms, q = ops._sm_count(torch.device(DEV)), lambda n: torch.zeros(n, 8 * 64, dtype=torch.bfloat16, device=DEV)
    cache, table = torch.zeros(plain_shape(400, 1, 16, 64), dtype=torch.uint8, device=DEV), torch.arange(400, dtype=torch.int32, device=DEV).view(1, 400)
    for tokens, want in ((4 * sms, []), (4 * sms + 1, [(0, 1)])):         # 16 rows a block, 8 heads a token, two blocks an SM
        ops.kv4_attention(q(tokens), q(tokens), cache, plain.make_step([0], [tokens], DEV), table, 0, 0.125, 8, 1, 64)
        assert calls == want


@pytest.mark.parametrize("n,batch", [(5000, 1), (2500, 3), (9000, 2)])
def test_many_keys(ops, n, batch):
    """Long enough for every way in which a sequence's keys are shared out; small heads keep the statement quick."""
    check(ops, torch.bfloat16, 4, 2, 64, 64, [n - 37 * s for s in range(batch)], [1] * batch, 0, True, 90)
    check(ops, torch.bfloat16, 4, 2, 64, 64, [n - 37 * s for s in range(batch)], [2] + [1] * (batch - 1), 0, False, 91)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,nkv,window", [(150, 4, 0), (150, 4, 700), (40, 2, 0), (33, 1, 0), (300, 2, 0), (9, 1, 0)])
@pytest.mark.parametrize("more", [0, 2])
def test_long_sequences_among_many_short_ones(ops, dtype, batch, nkv, window, more):
    """A few sequences are cut and the others are not; `more` further tokens in some."""
    longer = {0: 5000, batch // 2: 3100, batch - 1: 2500}
    starts = [longer.get(s, 1 + 37 * s % 90) for s in range(batch)]
    check(ops, dtype, 2 * nkv, nkv, 32, 32, starts, [1 + (more if s % 7 == 3 else 0) for s in range(batch)], window, False, 130)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_blocks_of_rows_than_a_launch_takes(ops, dtype):
    """A long portion beside single tokens whose blocks, counted by the longest, are more than 65,535."""
    check(ops, dtype, 64, 1, 32, 32, [40] * 7 + [0], [1] * 7 + [1200], 100, False, 140)


def test_a_pool_past_32_bits(ops):
    """Pages whose byte offsets, and whose rows read back, need more than 32 bits."""
    nkv, d, page = 8, 128, 16
    unit = nkv * 18 * d
    pages = (1 << 32) // unit + 50
    cache = torch.zeros(pages, nkv, 1, 18 * d, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[pages - 1, 3, pages - 7]], dtype=torch.int32, device=DEV)
    k, v = (random_rows(40, nkv, d, torch.bfloat16, s) for s in (1, 2))
    ops.kv4_write(k.to(DEV), v.to(DEV), plain.make_step([0], [40], DEV), table, cache)
    kept = [plain.kept(x)[2] for x in (k, v)]
    # a pool of read-back pages of over 2^32 bytes too
    out = [torch.empty((1 << 31) // (nkv * page * d) + 40, nkv, page, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    last = out[0].shape[0] - 1
    to = torch.tensor([[last, 0, last - 1]], dtype=torch.int32, device=DEV)
    ops.kv4_read(cache, table, torch.tensor([40], dtype=torch.int32, device=DEV), to, *out)
    for x, w in zip(out, kept):
        got = torch.cat([x[last], x[0], x[last - 1]], dim=1)[:, :40].cpu()
        assert torch.equal(got, w.bfloat16().transpose(0, 1))
    q = torch.randn(1, 32 * d, generator=torch.Generator().manual_seed(3)).bfloat16()
    o = torch.zeros(1, 32 * d, dtype=torch.bfloat16, device=DEV)
    ops.kv4_attention(q.to(DEV), o, cache, plain.make_step([39], [1], DEV), table, 0, d ** -0.5, 32, nkv, d)
    small = cache[[pages - 1, 3, pages - 7]]
    want, _ = plain.attention(q, small, torch.tensor([[0, 1, 2]]), [39], [1], 0, d ** -0.5, 32, nkv)
    top = max(float(x.abs().max()) for x in kept)
    assert bool(((o.cpu().double() - want).abs() <= 2.0 ** -8 * (want.abs() + top)).all())


@pytest.mark.parametrize("lens", [[1] * 5, [1, 1, 20, 7, 1]])
def test_same_bits_twice_and_on_another_stream(ops, lens):
    starts = [3, 800, 100, 411, 2000]
    kv = [a + n for a, n in zip(starts, lens)]
    cache, table = filled(kv, 2, 64, 32, torch.bfloat16, 95)
    q = torch.randn(sum(lens), 8 * 64, generator=torch.Generator().manual_seed(4)).bfloat16().to(DEV)
    step, outs = plain.make_step(starts, lens, DEV), []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), side, side, torch.cuda.current_stream()):
        with torch.cuda.stream(stream):
            o = torch.zeros_like(q)
            ops.kv4_attention(q, o, cache, step, table, 0, 0.125, 8, 2, 64)
        stream.synchronize()
        outs.append(o)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("lens", [[1] * 3, [70, 60, 2]])
def test_two_streams_at_once(ops, unpacked, lens):
    """Calls on two streams share nothing: neither the records of shared keys nor the unpacked ones."""
    starts = [6000, 4100, 30]
    cache, table = filled([a + n for a, n in zip(starts, lens)], 2, 64, 32, torch.bfloat16, 97)
    step, streams = plain.make_step(starts, lens, DEV), [torch.cuda.Stream() for _ in range(2)]
    qs = [torch.randn(sum(lens), 8 * 64, generator=torch.Generator().manual_seed(s)).bfloat16().to(DEV) for s in (5, 6)]
    run = lambda q, o: ops.kv4_attention(q, o, cache, step, table, 0, 0.125, 8, 2, 64)
    alone = [torch.zeros_like(q) for q in qs]
    for q, o in zip(qs, alone):
        run(q, o)
    outs = [[torch.zeros_like(q) for _ in range(20)] for q in qs]
    torch.cuda.synchronize()
    for i in range(20):
        for s, q, o in zip(streams, qs, outs):
            with torch.cuda.stream(s):
                run(q, o[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, a) for os, a in zip(outs, alone) for o in os)


def test_refusals(ops):
    E = ops.KernelError
    cache = torch.zeros(4, 2, 1, 18 * 64, dtype=torch.uint8, device=DEV)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    step = plain.make_step([3], [2], DEV)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device=DEV)
    bad = [
        lambda: ops.kv4_write(k, k.float(), step, table, cache),
        lambda: ops.kv4_write(k, k[:, :1], step, table, cache),
        lambda: ops.kv4_write(k.half(), k.half(), step, table, cache),
        lambda: ops.kv4_write(k.transpose(1, 2), k.transpose(1, 2), step, table, cache),
        lambda: ops.kv4_write(k[:1], k[:1], step, table, cache),
        lambda: ops.kv4_write(k, k, step, table.long(), cache),
        lambda: ops.kv4_write(k, k, step, table, cache[:, :1]),
        lambda: ops.kv4_write(k, k, step, table, cache.to(torch.int8)),
        lambda: ops.kv4_write(k.cpu(), k.cpu(), step, table, cache),
        lambda: ops.kv4_attention(q, q.float(), cache, step, table, 0, 1.0, 8, 2, 64),
        lambda: ops.kv4_attention(q, torch.zeros_like(q), cache, step, table, 0, 1.0, 7, 2, 64),
        lambda: ops.kv4_attention(q, torch.zeros_like(q), cache, step, table, 0, 1.0, 8, 2, 32),
        lambda: ops.kv4_attention(q[:1], torch.zeros_like(q[:1]), cache, step, table, 0, 1.0, 8, 2, 64),
        lambda: ops.kv4_attention(q, torch.zeros_like(q), cache, step, table, 0, 1.0, 8, 2, 64, sink=torch.zeros(7, device=DEV)),
        lambda: ops.kv4_attention(q, torch.zeros_like(q), cache, step, torch.zeros(2, 2, dtype=torch.int32, device=DEV), 0, 1.0, 8, 2, 64),
    ]
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    n = torch.tensor([5], dtype=torch.int32, device=DEV)
    bad += [
        lambda: ops.kv4_read(cache, table, n, table, pages, pages.float()),
        lambda: ops.kv4_read(cache, table, n, table[:, :1], pages, pages.clone()),
        lambda: ops.kv4_read(cache, table, torch.cat([n, n]), table, pages, pages.clone()),
        lambda: ops.kv4_read(cache, table, n, table, pages[:, :, :8].contiguous(), pages[:, :, :8].contiguous()),
        lambda: ops.kv4_cache_shape(4, 2, 8, 64),
        lambda: ops.kv4_cache_shape(4, 2, 16, 48),
        lambda: ops.kv4_cache_shape(4, 2, 16, 544),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(E):
            call()
            pytest.fail(f"call {i} was not refused")
    # nothing to do is no error
    empty = plain.make_step([3], [0], DEV)
    ops.kv4_write(k[:0], k[:0], empty, table, cache)
    ops.kv4_attention(q[:0], q[:0].clone(), cache, empty, table, 0, 1.0, 8, 2, 64)
