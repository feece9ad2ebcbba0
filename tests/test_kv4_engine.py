"""What the engine makes of a cache in 4 bits before any device is asked: needs, pages, refusals."""
import json
import os

import pytest
import torch

from helpers import CONFIGS
from inferloop_b200.cache.manager import CacheManager
from inferloop_b200.config.registry import read_model_config
from inferloop_b200.engine.runner import parse_kv_cache
from inferloop_b200.models.decoder import DecoderModel
from inferloop_b200.parts.base import BuildContext, CacheNeeds, PagedKVNeed, Workspace


def needs(name, kv_bits):
    _, _, spec = read_model_config(json.dumps(CONFIGS[name][0]))
    return DecoderModel(spec, BuildContext(torch.bfloat16, None, Workspace(None), kv_bits=kv_bits)).cache_needs()


def test_names():
    assert parse_kv_cache("auto") is None and parse_kv_cache("int4") == 4
    for bad in ("int8", "", None, 4, ["int4"]):
        with pytest.raises(ValueError, match="auto or int4"):
            parse_kv_cache(bad)


def test_pages_of_the_groups():
    for name in ("D", "E"):
        wide, four = (CacheManager(needs(name, bits), 16, 8, 2) for bits in (None, 4))
        assert [g.layers for g in wide.groups] == [g.layers for g in four.groups]
        for a, b in zip(wide.groups, four.groups):
            # 4.5 bits an element against 16
            assert b.page_bytes(2) * 32 == a.page_bytes(2) * 9 and b.need.bits == 4 and b.need.window == a.need.window
        assert [g["bits"] for g in four.inspect()["groups"]] == [4] * len(four.groups)


@pytest.mark.parametrize("need,page", [
    (PagedKVNeed(2, 64, bits=4), 8), (PagedKVNeed(2, 48, bits=4), 16), (PagedKVNeed(2, 64, v_head_dim=32, bits=4), 16),
    (PagedKVNeed(2, 544, bits=4), 16), (PagedKVNeed(2, 64, stride=16, bits=4), 16), (PagedKVNeed(2, 64, bits=8), 16)])
def test_geometries_that_no_cache_is_made_of(need, page):
    with pytest.raises(ValueError, match="4 bits"):
        CacheManager([CacheNeeds(paged=need)], page, 4, 2)


def test_layers_that_are_not_served():
    with pytest.raises(ValueError, match="4 bits"):
        needs("C", 4)                       # heads of 48
    with pytest.raises(ValueError, match="not served"):
        needs("D", 8)


def test_the_command_line_knows_it():
    from inferloop_b200.cli import build_parser
    from inferloop_b200.engine.trace import build_parser as trace_parser
    args = build_parser().parse_args(["generate", "/m", "--tokens", "1", "--kv-cache", "int4"])
    assert args.kv_cache == "int4"
    assert trace_parser().parse_args(["--model", "m", "--dtype", "bfloat16", "--out", "o", "--max-tokens", "64"]).kv_cache == "auto"
