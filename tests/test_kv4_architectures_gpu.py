"""A cache in 4 bits under the architectures beside the first that take it: heads' gates and biases next to a linear attention (Zebivik), interleaved
rotation with an unweighted norm behind it, under several residual streams and none (Sufolix).

The plain model attends to the rows that the engine's cache holds, so that no code on either side of a half comes in; those rows are held to the
plain model's own keys and values: half a step of the largest scale a group may have, (1 + 2^-8) / 7 of its largest element, and what the engine's
keys are off by.  Logits in 32 bits: attention is off by 2^-20 x 20 of the largest value, some five times a typical one: 1e-4 of the
largest logit; in bfloat16 the bound of every other engine test."""
import pytest
import torch

import kv4_plain
import plain_sufolix
import plain_zebivik
import sufolix_cases
import zebivik_cases
from helpers import assert_close, random_tokens

pytestmark = pytest.mark.gpu

_S = dict(heads=4, kv_heads=2, scale=0.12)
SUFOLIX = {
    "V": (sufolix_cases.model(500, 128, 1e-6, 1.0, 2, [
        sufolix_cases.layer(sufolix_cases.attention(rot=(10000.0, 128), v_mix=False, dim=128, vdim=128, **_S), sufolix_cases.dense(128)),
        sufolix_cases.layer(sufolix_cases.attention(rot=(500.0, 64), v_mix=False, dim=128, vdim=128, **_S), sufolix_cases.dense(192))]), 21, 16),
    "W": (sufolix_cases.model(300, 64, 1e-5, 2.0, None, [
        sufolix_cases.layer(sufolix_cases.attention(rot=(10000.0, 32), v_mix=False, dim=64, vdim=64, **_S), sufolix_cases.dense(96)),
        sufolix_cases.layer(sufolix_cases.attention(rot=None, v_mix=False, dim=64, vdim=64, **_S), None)]), 22, 32),
}


@pytest.fixture(scope="module")
def root(tmp_path_factory):
    return str(tmp_path_factory.mktemp("kv4_architectures"))


def run_plan(r, vocab):
    """request -> (tokens, logits) of two requests taken through portions, mixed steps and recorded single tokens."""
    from inferloop_b200.csrc import ops
    from inferloop_b200.engine.batch import StepEntry
    tokens = {"a": random_tokens(110, vocab, 1), "b": random_tokens(61, vocab, 2)}
    plan = [[("a", 60)], [("a", 1), ("b", 40)], [("a", 30), ("b", 1)], [("a", 3), ("b", 7)]] + [[("a", 1), ("b", 1)]] * 12 + [[("a", 1)]] * 4
    at, got = {"a": 0, "b": 0}, {"a": [], "b": []}
    for step in plan:
        logits, row = r.step([StepEntry(k, tokens[k][at[k]:at[k] + n], list(range(n))) for k, n in step]).clone(), 0
        for k, n in step:
            got[k].append(logits[row:row + n].cpu())
            row, at[k] = row + n, at[k] + n
    ops.check_device_errors()
    return {k: (tokens[k][:at[k]], torch.cat(got[k])) for k in tokens}


def check(folder, dtype, page, vocab, layers, forward, use, name):
    """`use(held)`: from then on the plain model's layers take their keys and values from the list."""
    from inferloop_b200.engine.runner import ModelRunner
    r = ModelRunner.from_folder(folder, dtype=dtype, page_size=page, num_pages=64, max_requests=4, kv_cache="int4")
    assert [len(g.layers) for g in r.cache.groups] == [layers] and r.cache.groups[0].storage.dtype == torch.uint8
    for request, (tokens, got) in run_plan(r, vocab).items():
        pages, held, own = r.cache.block_table(0, request), [], []
        for layer in range(layers):
            rows = kv4_plain.rows(r.cache.groups[0].storage[layer].cpu(), pages)
            held.append([x.transpose(1, 2).flatten(0, 1)[:len(tokens)] for x in rows])
        use(list(held), own)
        ref = forward(tokens)
        if dtype == "float32":
            assert bool(torch.isfinite(got).all()) and float((got.double() - ref).abs().max()) <= 1e-4 * float(ref.abs().max())
        else:
            assert_close(got, ref, dtype, f"{name} {request}")
        assert len(own) == layers
        off = 1e-5 if dtype == "float32" else 2e-2
        for mine, theirs in zip(held, own):
            for x, y in zip(mine, theirs):
                step = y.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1) * (1 + 2.0 ** -8) / 7
                assert bool(((x - y).abs() <= 0.5 * step + off * float(y.abs().max())).all())


@pytest.mark.parametrize("rounds", [0, 2])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_zebivik(root, monkeypatch, dtype, rounds):
    from inferloop_b200.csrc import ops
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", rounds)
    config, _, page = zebivik_cases.CASES["P"]
    stored = torch.float32 if dtype == "float32" else torch.bfloat16
    folder, model = zebivik_cases.folder(root, "P", stored), zebivik_cases.plain_model(root, "P", stored)

    def use(held, own):
        def attention(w, p, m, h, positions):
            T, H, G, d = h.shape[0], int(m["heads"]), int(m["kv_heads"]), int(m["dim"])
            q = (h @ w[p + "q"].T + w[p + "q.b"]).view(T, H, d)
            k = (h @ w[p + "k"].T + w[p + "k.b"]).view(T, G, d)
            v = (h @ w[p + "v"].T + w[p + "v.b"]).view(T, G, d)
            q, k = (plain_zebivik.rotate_half(x, positions, m["rot"]) for x in (q, k))
            own.append((k, v))
            k, v = held.pop(0)
            o = plain_sufolix.causal_attention(q, k, v, float(m["scale"])) * torch.sigmoid(h @ w[p + "g"].T)[:, :, None]
            return o.reshape(T, H * d) @ w[p + "o"].T + w[p + "o.b"]
        monkeypatch.setattr(plain_zebivik, "softmax_attention", attention)
    check(folder, dtype, page, config["vocab"], 1, model.forward, use, "Zebivik P")


@pytest.mark.parametrize("rounds", [0, 2])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["V", "W"])
def test_sufolix(root, monkeypatch, name, dtype, rounds):
    from inferloop_b200.csrc import ops
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", rounds)
    monkeypatch.setitem(sufolix_cases.CASES, name, SUFOLIX[name])
    config, _, page = SUFOLIX[name]
    stored = torch.float32 if dtype == "float32" else torch.bfloat16
    folder, model = sufolix_cases.folder(root, name, stored), sufolix_cases.plain_model(root, name, stored)
    attend = plain_sufolix.causal_attention

    def use(held, own):
        monkeypatch.setattr(plain_sufolix, "causal_attention", lambda q, k, v, scale: (own.append((k, v)), attend(q, *held.pop(0), scale))[1])
    check(folder, dtype, page, config["vocab"], 2, model.forward, use, f"Sufolix {name}")


@pytest.mark.parametrize("kv_cache", ["int4"])
def test_generation(root, kv_cache):
    from inferloop_b200 import Engine, SamplingParams
    config, _, page = zebivik_cases.CASES["P"]
    e = Engine(zebivik_cases.folder(root, "P", torch.bfloat16), dtype="bfloat16", block_size=page, num_gpu_blocks_override=64, max_num_seqs=4,
               prefill_chunk_tokens=64, kv_cache=kv_cache)
    got = e.generate([random_tokens(n, config["vocab"], 50 + n) for n in (5, 70, 130)], SamplingParams(), max_new_tokens=12)
    assert all(len(g) == 12 and all(0 <= t < config["vocab"] for t in g) for g in got)
    groups = e.runner.cache.inspect()["groups"]
    assert all(g["bits"] == 4 and g["free"] == g["total"] for g in groups)
