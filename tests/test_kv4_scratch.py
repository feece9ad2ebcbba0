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
