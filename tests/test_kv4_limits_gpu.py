"""What the 4-bit cache's operators do with tokens, tables and tensors at the edge of what they take: nothing is read or written outside them."""
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


def randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("before", [1, 3, 15, 16, 17, 31, 32, 33, 1000])
@pytest.mark.parametrize("dtype,off,mode", [(torch.bfloat16, 0, 0), (torch.bfloat16, 1, 0), (torch.bfloat16, 0, 1), (torch.float32, 0, 0)])
def test_tokens_before_the_first_position_are_left_out(ops, before, dtype, off, mode):
    """Rows of padding, at positions below 0, in every form of the input stage and of the write."""
    nq, nkv, d, page = 4, 2, 64, 32
    step = plain.make_step([5, 0], [2, 3], DEV)
    step.positions[2:4] = -before
    table = torch.tensor([[1, 2], [0, 3]], dtype=torch.int32, device=DEV)
    qkv = randn(5, (nq + 2 * nkv) * d + 8, seed=1).to(dtype).to(DEV)[:, off:off + (nq + 2 * nkv) * d]
    cache, want = (torch.zeros(6, nkv, page // 16, 18 * d, dtype=torch.uint8, device=DEV) for _ in range(2))
    cache[:2] = want[:2] = 0xA5                     # (what lies before page 0 of the cache that the call gets)
    q = torch.zeros(5, nq * d, dtype=dtype, device=DEV)
    ops.qk_norm_rope_kv4(qkv, q, None, None, 1e-6, None, 0, step, table, cache[2:], True, nq, nkv, d, mode)
    rows = qkv.unflatten(1, (-1, d)).cpu()
    pages = [(s, p) for s, p in zip(step.seq_of_token.tolist(), step.positions.tolist())]
    live = [i for i, (_, p) in enumerate(pages) if p >= 0]
    host = want.cpu()[2:].clone()
    plain.write(host, [int(table[pages[i][0], pages[i][1] // page]) for i in live], [pages[i][1] % page for i in live], rows[live, nq:nq + nkv], rows[live, nq + nkv:])
    assert bool((cache[:2] == 0xA5).all()) and torch.equal(cache[2:].cpu(), host)
    cache[2:] = 0
    ops.kv4_write(qkv.unflatten(1, (-1, d))[:, nq:nq + nkv], qkv.unflatten(1, (-1, d))[:, nq + nkv:], step, table, cache[2:])
    assert bool((cache[:2] == 0xA5).all()) and torch.equal(cache[2:].cpu(), host)


def requests(kv, nkv, d, page, seed):
    """(cache, block table) of sequences of so many keys."""
    table, pool = plain.make_table(kv, page, 2, seed)
    cache = torch.zeros(pool, nkv, page // 16, 18 * d, dtype=torch.uint8)
    for s, n in enumerate(kv):
        at = torch.arange(n)
        plain.write(cache, table[s, at // page], at % page, *(randn(n, nkv, d, seed=seed + 2 * s + i).bfloat16() for i in (0, 1)))
    return cache.to(DEV), table.to(DEV)


@pytest.mark.parametrize("window", [0, 700, -512])
@pytest.mark.parametrize("before", [1, 40, 1000000])
def test_queries_before_the_first_position_see_nothing(ops, window, before):
    """A row of padding beside long sequences whose keys are shared out: zeros, and the others as if it were not there, also in the calls after."""
    nq, nkv, d, kv = 8, 8, 32, [9000, 9000, 33, 9000]
    cache, table = requests(kv, nkv, d, 64, 7)
    q = randn(4, nq * d, seed=8).bfloat16()
    ref, bound = kv4_bounds.outcome(q, cache, table, [n - 1 for n in kv], [1] * 4, window, 0.2, nq, nkv)
    step = plain.make_step([n - 1 for n in kv], [1] * 4, DEV)
    for padded in (True, False, True):
        step.positions[2] = -before if padded else kv[2] - 1
        out = torch.full((4, nq * d), 5.0, dtype=torch.bfloat16, device=DEV)
        ops.kv4_attention(q.to(DEV), out, cache, step, table, window, 0.2, nq, nkv, d)
        rows = [0, 1, 3] if padded else [0, 1, 2, 3]
        assert bool(((out.cpu().double() - ref).abs() <= bound)[rows].all()) and not (padded and bool(out[2].any()))


@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("columns", [40, 1])
def test_keys_past_the_block_table_are_not_held(ops, monkeypatch, tokens, columns):
    """A length beyond the table's columns, by the codes and with every long portion unpacked."""
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", 0)
    nq, nkv, d, L = 8, 2, 64, 1000
    cache, table = requests([L], nkv, d, 16, 9)
    q = randn(tokens, nq * d, seed=10).bfloat16()
    known = table.clone()
    known[:, columns:] = -1
    ref, bound = kv4_bounds.outcome(q, cache, known, [L - tokens], [tokens], 0, 0.1, nq, nkv, unpacked=tokens > 1)
    out = torch.full((tokens, nq * d), 5.0, dtype=torch.bfloat16, device=DEV)
    ops.kv4_attention(q.to(DEV), out, cache, plain.make_step([L - tokens], [tokens], DEV), table[:, :columns].contiguous(), 0, 0.1, nq, nkv, d)
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_cache_off_its_boundary(ops, dtype):
    """On any even address attention is served; on an odd one it is refused, before anything runs."""
    nq, nkv, d, kv = 4, 2, 64, [33, 70]
    cache, table = requests(kv, nkv, d, 16, 11)
    q, step = randn(2, nq * d, seed=12).to(dtype).to(DEV), plain.make_step([n - 1 for n in kv], [1, 1], DEV)
    ref, bound = kv4_bounds.outcome(q, cache, table, [n - 1 for n in kv], [1, 1], 0, 0.1, nq, nkv)
    room = torch.zeros(cache.numel() + 16, dtype=torch.uint8, device=DEV)
    for off in (2, 8, 14, 1, 15):
        moved = room[off:off + cache.numel()].view(cache.shape)
        moved.copy_(cache)
        out = torch.full_like(q, 5.0)
        if off % 2:
            with pytest.raises(ops.KernelError, match="2-byte boundary"):
                ops.kv4_attention(q, out, moved, step, table, 0, 0.1, nq, nkv, d)
            assert bool((out == 5.0).all())
        else:
            ops.kv4_attention(q, out, moved, step, table, 0, 0.1, nq, nkv, d)
            assert bool(((out.cpu().double() - ref).abs() <= bound).all())


def test_steps_that_contradict_themselves(ops):
    """Fewer tokens than sequences in a step of single tokens, lengths of other sequences than it has, indices of other tokens: refused on the host."""
    nq, nkv, d = 4, 2, 64
    cache, table = requests([40, 40, 40], nkv, d, 16, 13)
    q = randn(3, nq * d, seed=14).bfloat16().to(DEV)

    def step(lens, **changes):
        st = plain.make_step([20] * len(lens), lens, DEV)
        for name, value in changes.items():
            setattr(st, name, value)
        return st
    call = lambda st, t, d=d, cache=cache: ops.kv4_attention(q[:t, :nq * d].contiguous(), torch.zeros(t, nq * d, dtype=q.dtype, device=DEV), cache, st, table,
                                                              0, 0.1, nq, nkv, d)
    call(step([1, 1, 1]), 3)
    call(step([0, 2, 1]), 3)
    bad = [(step([1, 1, 0], decode_only=True), 2), (step([0, 2, 1], kv_len=torch.zeros(2, dtype=torch.int32, device=DEV)), 3),
           (step([1, 1, 1], kv_len=torch.zeros(4, dtype=torch.int32, device=DEV)), 3), (step([0, 2, 1], h_q_len=[2, 1]), 3), (step([0, 2, 1], h_kv_len=[2, 1]), 3)]
    for st, t in bad:
        with pytest.raises(ops.KernelError, match="say otherwise"):
            call(st, t)
    with pytest.raises(ops.KernelError, match="do not agree"):           # no heads at all
        ops.kv4_attention(q, torch.zeros_like(q), cache[:, :0].contiguous(), step([1, 1, 1]), table, 0, 0.1, nq, 0, d)
    other = torch.zeros(3, nkv, 1, 18 * 160, dtype=torch.uint8, device=DEV)
    with pytest.raises(ops.KernelError, match="indices"):
        ops.kv4_attention(torch.zeros(3, nq * 160, device=DEV), torch.zeros(3, nq * 160, device=DEV), other,
                          step([1, 1, 1], seq_of_token=torch.zeros(2, dtype=torch.int32, device=DEV)), table, 0, 0.1, nq, nkv, 160)
