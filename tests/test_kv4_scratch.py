"""Scratch of portions over a cache in 4 bits: how it grows, what a recorded step notices of it, what a model's memory plan counts."""
import torch

from inferloop_b200.csrc import ops
from inferloop_b200.parts.base import Workspace


def test_buffers_of_steps_that_are_not_recorded():
    ws, f32 = Workspace(torch.device("cpu")), torch.float32
    at = ws.unrecorded("x", 10, f32, room=100)
    assert ws.nbytes() == 400 and ws.unrecorded("x", 100, f32, room=100) == at and ws.generation == 0
    ws.unrecorded("x", 101, f32, room=100)
    assert ws.nbytes() == 800 and ws.generation == 0                  # by doubling
    ws.unrecorded("x", 1000, f32, room=100)
    assert ws.nbytes() == 4000 and ws.generation == 0
    ws.unrecorded("x", 1000, f32, room=2000)                          # another caller's room comes with its first call that needs it
    assert ws.nbytes() == 4000
    ws.unrecorded("x", 1001, f32, room=3000)
    assert ws.nbytes() == 12000 and ws.generation == 0
    at = ws.unrecorded("x", 5, f32, recording=True)                   # a recorded step holds the address from here on
    assert ws.generation == 0 and ws.unrecorded("x", 3000, f32) == at
    ws.unrecorded("x", 3001, f32)
    assert ws.generation == 1
    ws.address("y", 4, f32)
    assert ws.generation == 2


def test_room_of_unpacked_keys():
    assert ops.kv4_unpack_room(None) == ops.KV4_UNPACK_TOKENS == ops.kv4_unpack_room(40960) == ops.kv4_unpack_room(10 ** 7)
    assert ops.kv4_unpack_room(2048) == 8 * 2048 and ops.kv4_unpack_room(130) == 8 * 256


def test_memory_that_a_model_plans_for():
    """Room for unpacked keys only where portions are unpacked, and for requests as long as they get."""
    bf16, f32, tokens = torch.bfloat16, torch.float32, 575
    plan = lambda dtype, d=128, longest=None: ops.kv4_scratch_bytes(tokens, 32, 8, d, dtype, longest)  # noqa: E731
    records = lambda d: (tokens * 8 + 12 * 148) * 8 * (d + 4) * 4  # noqa: E731   (blocks and further runs, of 8 rows of d sums, a maximum, a sum, and two more)
    assert plan(f32) == plan(f32, longest=2048) == records(128) and plan(bf16, 96) == records(96)
    unpacked = plan(bf16) - plan(f32)
    assert unpacked >= ops.KV4_UNPACK_TOKENS * 8 * 128 * 4
    assert plan(bf16, longest=40960) == plan(bf16) and plan(bf16, longest=2048) - plan(f32) < unpacked / 7


def test_layers_ask_for_their_model():
    """The plan of a whole model follows the cache's type, the compute type and the longest request."""
    import json
    from helpers import CONFIGS
    from inferloop_b200.config.registry import read_model_config
    from inferloop_b200.models.decoder import DecoderModel
    from inferloop_b200.parts.base import BuildContext
    _, _, spec = read_model_config(json.dumps(CONFIGS["D"][0]))

    def plan(dtype, bits, longest):
        ctx = BuildContext(dtype, None, Workspace(None), longest=longest, kv_bits=bits)
        return DecoderModel(spec, ctx).scratch_bytes(64, 4)
    nkv, d = CONFIGS["D"][0]["num_key_value_heads"], CONFIGS["D"][0]["head_dim"]
    whole = ops.KV4_UNPACK_TOKENS * nkv * d * 4
    four = {longest: plan(torch.bfloat16, 4, longest) - plan(torch.bfloat16, None, longest) for longest in (None, 2048)}
    assert four[None] > whole and four[2048] < whole / 4
    assert plan(torch.float32, 4, None) - plan(torch.float32, None, None) < 10 << 20
