"""Attention over the 4-bit cache in recorded graphs, by callers that bring no workspace of their own: what a recording reads is its own."""
import pytest
import torch

import kv4_plain as plain

pytestmark = pytest.mark.gpu
DEV, NQ, NKV, D, PAGE, SCALE = "cuda:0", 8, 2, 64, 16, 0.1
KINDS = [("shared keys", [1, 1], [6000, 900]), ("portions", [90, 1], [300, 20])]


@pytest.fixture
def ops(monkeypatch):
    from inferloop_b200.csrc import ops
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", 0)
    monkeypatch.setattr(ops, "_KV4_WORKSPACE", {})
    return ops


def call_of(ops, lens, kv, seed):
    """(a call, its output, what the call gives outside a recording)."""
    gen = torch.Generator().manual_seed(seed)
    table, pool = plain.make_table(kv, PAGE, 2, seed)
    cache = torch.randint(0, 256, (pool, NKV, 1, 18 * D), dtype=torch.uint8, generator=gen)
    cache[..., 16 * D:] = torch.rand(pool, NKV, 1, D, generator=gen).bfloat16().view(torch.uint8)
    q = torch.randn(sum(lens), NQ * D, generator=gen).bfloat16().to(DEV)
    cache, table, step, out = cache.to(DEV), table.to(DEV), plain.make_step([n - k for n, k in zip(kv, lens)], lens, DEV), torch.empty_like(q)
    call = lambda: ops.kv4_attention(q, out, cache, step, table, 0, SCALE, NQ, NKV, D)  # noqa: E731
    call()
    torch.cuda.synchronize()
    want = out.clone()
    assert bool(torch.isfinite(want).all()) and float(want.float().abs().max()) > 0.1
    return call, out, want


def recorded(call, stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    return graph


def replayed(graph, out, want):
    out.fill_(5.0)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    return torch.equal(out, want)


@pytest.mark.parametrize("name,lens,kv", KINDS)
def test_recordings_replayed_out_of_order(ops, name, lens, kv):
    """Two recordings on a stream that has seen no call: the second does not lean on what the first sets up when it is replayed."""
    side = torch.cuda.Stream()
    first, second = (call_of(ops, lens, kv, s) for s in (1, 2))
    graphs = [recorded(c[0], side) for c in (first, second)]
    for ws in [w for (_, stream), w in ops._KV4_WORKSPACE.items() if stream == side.cuda_stream]:
        for buffer in ws._buffers.values():
            buffer.fill_(3)                       # what nothing has been written to may hold anything
    assert replayed(graphs[1], *second[1:]) and replayed(graphs[0], *first[1:]) and replayed(graphs[1], *second[1:])


@pytest.mark.parametrize("name,lens,kv", KINDS)
def test_a_larger_call_between_recording_and_replay(ops, name, lens, kv):
    """A recording made after a warm-up call on its stream keeps what it reads when a larger call on that stream grows the stream's buffers."""
    side = torch.cuda.Stream()
    call, out, want = call_of(ops, lens, kv, 3)
    large, large_out, large_want = call_of(ops, [3 * n for n in lens] if max(lens) > 1 else lens * 40, [3 * n for n in kv] if max(lens) > 1 else kv * 40, 4)
    with torch.cuda.stream(side):
        call()
        graph = recorded(call, side)
        kept = [b for w in ops._KV4_WORKSPACE.values() for b in w._buffers.values()] + [b for r in getattr(ops, "_KV4_RECORDS", {}).values() for b in r[4]]
        sizes = [b.numel() * b.element_size() for b in kept]
        del kept
        side.synchronize()
        large()
        side.synchronize()
        assert torch.equal(large_out, large_want)
        others = [torch.full((n // 4,), 0x7a7a7a7a, dtype=torch.int32, device=DEV) for n in sizes if n for _ in range(2)]
        side.synchronize()
    assert replayed(graph, out, want) and replayed(graph, out, want)
    assert all(bool((x == 0x7a7a7a7a).all()) for x in others)
