"""Long prompts beside recorded steps, over a cache in 4 bits."""
import pytest
import torch

from helpers import CONFIGS, random_tokens

pytestmark = pytest.mark.gpu


def test_recorded_steps_outlive_a_long_prompt(monkeypatch):
    """Steps of single tokens recorded before a prompt of 16,000 tokens are replayed after it, and its portions ask for scratch once."""
    from inferloop_b200.csrc import ops
    from inferloop_b200.engine.batch import StepEntry
    from inferloop_b200.engine.runner import ModelRunner
    monkeypatch.setattr(ops, "KV4_ROWS_ROUNDS", 0)
    cfg, chunk = dict(CONFIGS["D"][0], max_position_embeddings=17000), 500
    r = ModelRunner.from_config(cfg, 3, dtype="bfloat16", page_size=16, num_pages=1200, max_requests=4, kv_cache="int4")
    portions, inner, sizes = [], ops._kv4_portions, set()
    monkeypatch.setattr(ops, "_kv4_portions", lambda *args: (portions.append(1), inner(*args)))
    step = lambda request, tokens: r.step([StepEntry(request, tokens, [len(tokens) - 1])])  # noqa: E731
    step("a", random_tokens(chunk, cfg["vocab_size"], 1))
    for t in range(3):
        step("a", [t])
    recorded, replays = dict(r.graphs._recorded), r.graphs.replays
    assert recorded and replays >= 1 and portions
    for i in range(32):
        step("b", random_tokens(chunk, cfg["vocab_size"], 10 + i))
        sizes.add(r.ctx.workspace.nbytes())
    assert len(portions) >= 33 and len(sizes) == 1
    for t in range(3):
        assert bool(torch.isfinite(step("a", [t])).all())
    assert r.graphs.replays == replays + 3 and all(r.graphs._recorded[k] is rec for k, rec in recorded.items())
    ops.check_device_errors()
    asked = sum(b.numel() * b.element_size() for (tag, _), b in r.ctx.workspace._buffers.items() if tag.startswith("kv4."))
    assert asked <= ops.kv4_scratch_bytes(chunk, cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], torch.bfloat16, 17000)
