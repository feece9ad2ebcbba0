"""The engine over a cache in 4 bits against the plain model whose keys and values are kept as the definition says.

Tolerances.  A key or value whose quotient by its scale lies within the engine's own error of a half is kept a step away.  In the
32-bit engine that is some 1e-6 of the elements, one of which moves a logit by 1e-3 of the largest at most.  In the bfloat16 engine,
whose activations are off by 2^-9, it is some hundredths of them, a noise as large as that of keeping 4 bits at all: its logits are
held against the plain model over the rows that the engine's own cache holds, to the bfloat16 bound of every other engine test."""
import pytest
import torch

import kv4_plain
import plain_qwen3 as plain
from helpers import CONFIGS, assert_close, make_model_folder, random_tokens

pytestmark = pytest.mark.gpu
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("kv4_models")
    return {n: make_model_folder(str(root / n), CONFIGS[n][0], CONFIGS[n][1]) for n in ("B", "D", "E", "F")}


@pytest.fixture
def kept_rows(monkeypatch):
    attend = plain.causal_attention
    monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, *rest: attend(q, kv4_plain.kept(k)[2], kv4_plain.kept(v)[2], *rest))


def run_plan(r, vocab):
    """(tokens, logits) of two requests taken through portions and single tokens."""
    from inferloop_b200.engine.batch import StepEntry
    assert r.cache.groups[0].storage.dtype == torch.uint8
    a, b = random_tokens(100, vocab, 1), random_tokens(61, vocab, 2)
    got_a, got_b = [], []
    # a whole portion, portions beside single tokens, single tokens alone (the recorded steps)
    plan = [[("a", 50)], [("a", 1), ("b", 40)], [("a", 30), ("b", 1)], [("a", 3), ("b", 7)]] + [[("a", 1), ("b", 1)]] * 12 + [[("a", 1)]] * 4
    at = {"a": 0, "b": 0}
    for step in plan:
        entries = [StepEntry(k, (a if k == "a" else b)[at[k]:at[k] + n], list(range(n))) for k, n in step]
        logits = r.step(entries).clone()
        row = 0
        for k, n in step:
            (got_a if k == "a" else got_b).append(logits[row:row + n].cpu())
            row, at[k] = row + n, at[k] + n
    from inferloop_b200.csrc import ops
    ops.check_device_errors()
    return {"a": (a[:at["a"]], torch.cat(got_a)), "b": (b[:at["b"]], torch.cat(got_b))}


@pytest.mark.parametrize("name", ["B", "D", "E", "F"])
def test_logits_of_prompts_portions_and_single_tokens(folders, kept_rows, name):
    from inferloop_b200.engine.runner import ModelRunner
    r = ModelRunner.from_folder(folders[name], dtype="float32", page_size=16, num_pages=64, max_requests=4, kv_cache="int4")
    model = plain.PlainModel(folders[name])
    for tokens, got in run_plan(r, CONFIGS[name][0]["vocab_size"]).values():
        ref = model.logits(tokens)
        assert bool(torch.isfinite(got).all())
        assert float((got.double() - ref).abs().max()) <= 1e-3 * float(ref.abs().max())


@pytest.mark.parametrize("name", ["B", "D", "F"])
def test_logits_over_the_rows_that_the_cache_holds(folders, monkeypatch, name):
    from inferloop_b200.engine.runner import ModelRunner
    r = ModelRunner.from_folder(folders[name], dtype="bfloat16", page_size=16, num_pages=64, max_requests=4, kv_cache="int4")
    model = plain.PlainModel(folders[name], round_to_bf16=True)
    attend = plain.causal_attention
    for request, (tokens, got) in run_plan(r, CONFIGS[name][0]["vocab_size"]).items():
        pages, held = r.cache.block_table(0, request), []
        for layer in range(CONFIGS[name][0]["num_hidden_layers"]):
            rows = kv4_plain.rows(r.cache.groups[0].storage[layer].cpu(), pages)
            held.append([x.transpose(1, 2).flatten(0, 1)[:len(tokens)] for x in rows])
        monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, *rest: attend(q, *held.pop(0), *rest))
        assert_close(got, model.logits(tokens), "bfloat16", f"{name} {request}")
        assert not held


def test_logits_with_every_long_portion_unpacked(folders, monkeypatch):
    from inferloop_b200.csrc import ops
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", 0)
    calls, inner = [], ops._kv4_portions
    monkeypatch.setattr(ops, "_kv4_portions", lambda *args: (calls.append(1), inner(*args)))
    test_logits_over_the_rows_that_the_cache_holds(folders, monkeypatch, "D")
    assert calls


@pytest.mark.parametrize("name", ["B", "D"])
def test_generation_and_pages_given_back(folders, kept_rows, name):
    from inferloop_b200 import Engine, SamplingParams
    engine = Engine(folders[name], dtype="float32", block_size=16, num_gpu_blocks_override=40, max_num_seqs=4, prefill_chunk_tokens=32, kv_cache="int4")
    prompts = [random_tokens(n, CONFIGS[name][0]["vocab_size"], 30 + n) for n in (3, 40, 75)]
    got = engine.generate(prompts, SamplingParams(), max_new_tokens=10)
    model = plain.PlainModel(folders[name])
    for p, g in zip(prompts, got):
        ref = model.logits(p + g)[len(p) - 1:-1]
        bound = 1e-3 * float(ref.abs().max())
        assert len(g) == 10 and all(ref[i, t] >= ref[i].max() - 2 * bound for i, t in enumerate(g))
    groups = engine.runner.cache.inspect()["groups"]
    assert all(g["bits"] == 4 and g["free"] == g["total"] for g in groups)


def test_default_pool_holds_three_and_a_half_times_the_tokens(folders):
    from inferloop_b200 import Engine
    cfg = dict(CONFIGS["D"][0], max_position_embeddings=40000000)        # (no request's length bounds the pool)
    pages = []
    for kv in ("auto", "int4"):
        e = Engine(cfg, dtype="bfloat16", max_num_seqs=4, gpu_memory_utilization=0.05, random_weights_seed=1, kv_cache=kv, cuda_graphs=False)
        pages.append(e.runner.cache.groups[0].pool.num_pages)
        del e
        torch.cuda.empty_cache()
    assert pages[1] > 3 * pages[0]


def test_input_stage_keeps_what_the_write_keeps():
    """Queries as `qk_norm_rope_cache` makes them, values as `kv4_write` keeps them, keys a step away at most where the order of the norm's
    sum decides; every mode of the norm and the rotation."""
    from inferloop_b200.csrc import ops
    dev = "cuda:0"
    gen = torch.Generator().manual_seed(5)
    nq, nkv = 6, 2
    for d, rd, dtype in ((64, 64, torch.bfloat16), (128, 64, torch.float32), (96, 96, torch.bfloat16), (256, 128, torch.bfloat16), (32, 32, torch.float32)):
        for mode in (0, ops.ROPE_INTERLEAVED, ops.NORM_AFTER_ROTATION, ops.NORM_UNWEIGHTED | ops.ROPE_INTERLEAVED):
            starts, lens = [30, 0, 7], [1, 20, 3]
            step = kv4_plain.make_step(starts, lens, dev)
            table, pool = kv4_plain.make_table([a + n for a, n in zip(starts, lens)], 16, 1, 3)
            T = sum(lens)
            qkv = torch.randn(T, (nq + 2 * nkv) * d + 8, generator=gen).to(dtype).to(dev)
            weights = [None, None] if mode & ops.NORM_UNWEIGHTED else [(1 + 0.1 * torch.randn(d, generator=gen)).to(dev) for _ in range(2)]
            angle = torch.rand(T, rd // 2, generator=gen) * 6
            rope = torch.stack([angle.cos(), angle.sin()], -1).contiguous().to(dev)
            table = table.to(dev)
            wide = [torch.zeros(pool, nkv, 16, d, dtype=torch.float32, device=dev) for _ in range(2)]
            q_ref, q = (torch.zeros(T, nq * d, dtype=dtype, device=dev) for _ in range(2))
            ops.qk_norm_rope_cache(qkv, q_ref, *weights, 1e-6, rope, rd, step.positions, step.seq_of_token, table, 16, *wide, nq, nkv, d, mode=mode)
            cache, again = (torch.zeros(ops.kv4_cache_shape(pool, nkv, 16, d), dtype=torch.uint8, device=dev) for _ in range(2))
            ops.qk_norm_rope_kv4(qkv, q, *weights, 1e-6, rope, rd, step, table, cache, True, nq, nkv, d, mode)
            assert float((q.float() - q_ref.float()).abs().max()) <= 2.0 ** (-7 if dtype == torch.bfloat16 else -20) * float(q_ref.float().abs().max())
            v = qkv[:, (nq + nkv) * d:(nq + 2 * nkv) * d].unflatten(1, (nkv, d))
            k = torch.stack([wide[0][table[s, p // 16].long(), :, p % 16] for s, p in zip(step.seq_of_token.tolist(), step.positions.tolist())])
            ops.kv4_write(k.to(dtype), v, step, table, again)
            got, ref = kv4_plain.rows(cache.cpu(), list(range(pool))), kv4_plain.rows(again.cpu(), list(range(pool)))
            assert torch.equal(got[1], ref[1])
            rows = [(int(table[s, p // 16]), p % 16) for s, p in zip(step.seq_of_token.tolist(), step.positions.tolist())]
            for i, (page, slot) in enumerate(rows):
                _, scale, want = kv4_plain.kept(k[i].cpu())
                err = (got[0][page, :, slot] - want).abs().unflatten(-1, (-1, 32))
                assert bool((err <= 1.01 * scale[..., None]).all()) and float((err > 0.02 * scale[..., None]).float().mean()) < 0.02
            cache.zero_()
            ops.qk_norm_rope_kv4(qkv, q, *weights, 1e-6, rope, rd, step, table, cache, False, nq, nkv, d, mode)
            assert not bool(cache.any())


@pytest.mark.parametrize("d,nq,nkv", [(64, 9, 3), (128, 32, 8), (128, 5, 1), (64, 2, 2)])
@pytest.mark.parametrize("starts,lens", [([30, 0], [2, 1]), ([0, 17], [260, 41])])
@pytest.mark.parametrize("norm,turn", [(True, True), (False, True), (True, False), (False, False)])
def test_input_stage_in_vectors_is_the_general_one(d, nq, nkv, starts, lens, norm, turn):
    """Rows on 16-byte boundaries and off them, with one page not held.  Norms summed in another order are 2^-22 apart: queries a
    rounding to bfloat16, values nothing, keys a code or scale whose rounding hung on it (1e-3 of the bytes at the most)."""
    from inferloop_b200.csrc import ops
    dev, T, page = "cuda:0", sum(lens), 32
    gen = torch.Generator().manual_seed(6)
    step = kv4_plain.make_step(starts, lens, dev)
    table, pool = kv4_plain.make_table([a + n for a, n in zip(starts, lens)], page, 1, 3)
    table[0, 0] = -1
    table = table.to(dev)
    width = (nq + 2 * nkv) * d
    even = torch.randn(T, width + 8, generator=gen).to(torch.bfloat16).to(dev)
    odd = torch.zeros(T, width + 9, dtype=torch.bfloat16, device=dev)
    odd[:, 1:1 + width] = even[:, :width]
    weights = [(1 + 0.1 * torch.randn(d, generator=gen)).to(dev) if norm else None for _ in range(2)]
    angle = torch.rand(T, d // 2, generator=gen) * 6
    rope = torch.stack([angle.cos(), angle.sin()], -1).contiguous().to(dev) if turn else None
    found = []
    for qkv in (even[:, :width], odd[:, 1:1 + width]):
        q = torch.full((T, nq * d), 9.0, dtype=torch.bfloat16, device=dev)
        cache = torch.zeros(ops.kv4_cache_shape(pool, nkv, page, d), dtype=torch.uint8, device=dev)
        ops.qk_norm_rope_kv4(qkv, q, *weights, 1e-6, rope, d if turn else 0, step, table, cache, True, nq, nkv, d)
        found.append((q.double(), cache))
    (q, cache), (q_ref, ref) = found
    assert bool(((q - q_ref).abs() <= 2.0 ** -7 * q_ref.abs() + 2.0 ** -20).all())
    values = torch.zeros(18 * d, dtype=torch.bool, device=dev)
    values[8 * d:16 * d] = values[17 * d:] = True
    assert int(cache.sum()) > 0 and torch.equal(cache[..., values], ref[..., values])
    wrong = float((cache != ref).float().mean())
    assert wrong <= 1e-3 if norm else wrong == 0


def test_refusals_of_the_engine(folders):
    from inferloop_b200 import Engine
    with pytest.raises(ValueError, match="auto or int4"):
        Engine(folders["D"], kv_cache="int8", num_gpu_blocks_override=8)
    with pytest.raises(ValueError, match="multiple of 16"):
        Engine(folders["D"], kv_cache="int4", block_size=8, num_gpu_blocks_override=8)
