"""The 4-bit key/value cache: writing it, reading it back, attention over it, as cases that can be timed and checked.

The cache of a layer is a uint8 tensor [pages, kv_heads, page_size / 16, 18 d]: per page and kv head, units of 16 tokens, each
keys' codes (8 d bytes), values' codes (8 d), keys' scales (16 x d / 32 bfloat16), values' scales (the same).  32 neighbouring
elements of a row share a scale s = bfloat16(max |x| / 7) (0 below 2^-126); an element is c s with c = x / s rounded, halves away
from zero, stored as c + 8 in four bits.  Where a code lies:

  key   j, element 32 G + 8 t + i: nibble i of the 32-bit word at byte  j d / 2 + t d / 8 + 4 G
  value j, element 32 G + 4 g + i: nibble i of the 16-bit word at byte  ((j / 8) 32 + 4 g + (j / 2) % 4) d / 8 + (j % 2) d / 16 + 2 G

The kinds of pass:

  write    a step's new keys and values go into the cache, and the pages that they touch are read back
  read     whole requests are read back as pages of the compute type
  attend   the step's queries attend to everything that their requests have in the cache

Sizes are those of bench.py and of the tests: 32 / 8, 40 / 8 and 64 / 8 heads of 128 and small models with heads of 64 and 32.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False
DEVICE = "cuda:0"
UNIT = 16          # tokens of a unit
GROUP = 32         # elements that share a scale
F64 = torch.float64


def _case(name, kind, batch, context, tokens=1, nq=32, nkv=8, d=128, page=16, dtype="bfloat16", window=0, sink=False):
    """batch: requests of the step; context: tokens that the longest has in the cache before it; tokens: those it brings;
    window: keys that a token sees (0: all; negative: those of its aligned chunk); sink: a logit a head in the denominator."""
    c = dict(kind=kind, batch=batch, context=context, tokens=tokens, nq=nq, nkv=nkv, d=d, page=page, dtype=dtype, window=window, sink=sink)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user, one new token: the smallest call, a launch's latency
        _case("write 1 token", "write", 1, 70),
        # a busy server's decode step: a token of each of 64 requests, pages all over the pool
        _case("write 64 tokens", "write", 64, 1024),
        # a prompt's portion as the prefill writes it, then reads it for the attention
        _case("write portion 2048", "write", 1, 0, tokens=2048),
        # the 32-bit engine's portions of two requests, odd length, small heads
        _case("write float32 2 x 301", "write", 2, 45, tokens=301, nq=8, nkv=2, d=64, dtype="float32"),
        # one short conversation read back (before a portion of it is attended to)
        _case("read 1 x 333", "read", 1, 333),
        # eight long ones
        _case("read 8 x 6000", "read", 8, 6000, page=64),
        # one user's decode step: latency
        _case("attend 1 x 1030", "attend", 1, 1030),
        # the headline: 64 requests decoding together, ragged lengths
        _case("attend 64 x 1030", "attend", 64, 1030),
        # few long conversations, groups of eight heads
        _case("attend 2 x 16000", "attend", 2, 16000, nq=64),
        # the 32-bit engine, a window, a learned sink, small heads
        _case("attend float32 19 x 700", "attend", 19, 700, nq=8, nkv=2, d=64, dtype="float32", window=500, sink=True),
        # a short question behind a long document (its few tokens against all that is cached)
        _case("attend 7 tokens behind 7000", "attend", 1, 7000, tokens=7, nq=40),
        # a portion of a prompt behind its earlier ones
        _case("attend portion 1024 behind 1024", "attend", 1, 1024, tokens=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend"])
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    nkv = rng.choice([1, 2, 4, 8, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 4, 5, 8, 8, 12, 16])
    d = rng.choice([32, 64, 64, 96, 128, 128, 128, 256])
    page = rng.choice([16, 16, 16, 32, 64, 128])
    room = max(1, 1024 // (nkv * d))              # how many times the rows of 8 heads of 128 fit these
    if kind == "write":
        batch = _log(rng, 1, 100)
        tokens = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, 2048 // batch))
        return _case(None, kind, batch, _log(rng, 1, 600) - 1, tokens, nkv * group, nkv, d, page, dtype)
    if kind == "read":
        batch = _log(rng, 1, 24)
        return _case(None, kind, batch, _log(rng, 1, max(1, min(8000, 30000 * min(room, 2) // batch))), 1, nkv * group, nkv, d, page, dtype)
    window = rng.choice([0, 0, 0, 0, 40, 500, -256])
    sink = rng.random() < 0.2
    if rng.random() < 0.6:                        # single tokens
        batch = _log(rng, 1, 100)
        context = _log(rng, 1, max(1, min(30000, 60000 // batch))) - 1
        if dtype == "float32":
            context = min(context, 4000)
        return _case(None, kind, batch, context, 1, nkv * min(group, 8) if dtype == "float32" else nkv * group, nkv, d, page, dtype, window, sink)
    batch = _log(rng, 1, 6)
    tokens = _log(rng, 2, max(2, (128 if dtype == "float32" else 1024) // batch))
    context = _log(rng, 1, max(1, min(6000, 800000 // (tokens * batch)))) - 1
    group = min(group, max(1, 32 // nkv))
    return _case(None, kind, batch, context, tokens, nkv * group, nkv, d, page, dtype, window, sink)


# ------------------------------------------------------------------ lengths of the requests
def _lens(case):
    """(tokens brought, tokens in the cache afterwards) of each request: ragged, the first the longest."""
    new, kv = [], []
    for s in range(case["batch"]):
        n = max(1, case["tokens"] - (s * 29) % (case["tokens"] // 4 + 1))
        c = max(0, case["context"] - (s * 41) % (case["context"] // 4 + 1))
        if case["kind"] == "read":
            n, c = 0, max(1, c)
        new.append(n)
        kv.append(c + n)
    return new, kv


def _first_key(pos, window):
    return max(0, pos + 1 - window) if window > 0 else pos - pos % -window if window < 0 else 0


def _visible(case):
    """(keys read by some token of the step, pairs of token and key it sees), over all requests."""
    keys = pairs = 0
    for n, kv in zip(*_lens(case)):
        keys += kv - _first_key(kv - n, case["window"])
        pairs += sum(p + 1 - _first_key(p, case["window"]) for p in range(kv - n, kv))
    return keys, pairs


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    row = case["nkv"] * case["d"]                          # elements of a token's keys
    held = row * 9 // 8                                    # bytes of a token's keys and values in the cache
    new, kv = _lens(case)
    page = case["page"]
    if case["kind"] == "write":
        out = sum(-(-k // page) - (k - n) // page for n, k in zip(new, kv)) * page
        back = sum(k - (k - n) // page * page for n, k in zip(new, kv))
        return {"bytes": sum(new) * (2 * row * e + held) + back * held + out * 2 * row * e, "flops": 0}
    if case["kind"] == "read":
        return {"bytes": sum(kv) * held + sum(-(-k // page) for k in kv) * page * 2 * row * e, "flops": 0}
    keys, pairs = _visible(case)
    return {"bytes": keys * held + 2 * sum(new) * case["nq"] * case["d"] * e, "flops": 4 * pairs * case["nq"] * case["d"]}


# ------------------------------------------------------------------ the plain form
def _quantise(x):
    """Rows [..., d] -> codes -7..7 and scales, groups of 32, in 32 bits."""
    g = x.float().unflatten(-1, (-1, GROUP))
    amax = g.abs().amax(-1, keepdim=True)
    amax = torch.where(torch.isfinite(g).all(-1, keepdim=True), amax, torch.full_like(amax, float("nan")))
    s = (amax * torch.tensor(1.0 / 7.0, dtype=torch.float32, device=x.device)).to(torch.bfloat16).float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    y = g / torch.where(s == 0, torch.ones_like(s), s)
    y = torch.where((s == 0) | torch.isnan(s), torch.zeros_like(y), y)
    whole = torch.floor(y.abs())
    c = whole + (y.abs() - whole >= 0.5).float()
    return (torch.copysign(c, y).clamp(-7, 7), s.squeeze(-1).to(torch.bfloat16))


def _bytes(nibbles):
    n = (nibbles + 8).to(torch.uint8).unflatten(-1, (-1, 2))
    return n[..., 0] | (n[..., 1] << 4)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2).float() - 8


def _plain_write(k, v, pages, slots, cache):
    """k, v [T, nkv, d] into rows `slots` of pages `pages` of the cache."""
    T, nkv, d = k.shape
    gr = d // GROUP
    flat = cache.view(-1, cache.shape[-1])
    j = slots % UNIT
    unit = ((pages[:, None] * nkv + torch.arange(nkv, device=k.device)) * cache.shape[2] + (slots // UNIT)[:, None])[..., None]
    c, s = _quantise(k)
    at = torch.arange(d // 2, device=k.device)
    flat[unit, (j * (d // 2))[:, None, None] + at] = _bytes(c.view(T, nkv, gr, 4, 8).transpose(2, 3).flatten(2))
    at = torch.arange(d // 16, device=k.device)
    flat[unit, (16 * d + j * (d // 16))[:, None, None] + at] = s.contiguous().view(torch.uint8)
    c, s = _quantise(v)
    flat[unit, (17 * d + j * (d // 16))[:, None, None] + at] = s.contiguous().view(torch.uint8)
    piece = torch.arange(8, device=k.device)[:, None] * (d // 2) + at
    place = (8 * d + (j // 8) * (4 * d) + (j // 2 % 4) * (d // 8) + (j % 2) * (d // 16))[:, None, None] + piece.flatten()
    flat[unit, place] = _bytes(c.view(T, nkv, gr, 8, 4).transpose(2, 3).flatten(2))


def _plain_rows(cache, pages, d):
    """Keys and values [n, nkv, page, d] of the pages, in 32 bits."""
    u = cache[pages]                                       # [n, nkv, units, 18 d]
    gr, lead = d // GROUP, u.shape[:3]
    scale = u[..., 16 * d:].contiguous().view(torch.bfloat16).float().view(*lead, 2, UNIT, gr, 1)
    k = _nibbles(u[..., :8 * d]).view(*lead, UNIT, 4, gr, 8).transpose(4, 5).reshape(*lead, UNIT, gr, GROUP)
    # (half, piece, pair, which of the pair, group, element) -> (half, pair, which, group, piece, element)
    v = _nibbles(u[..., 8 * d:16 * d]).view(*lead, 2, 8, 4, 2, gr, 4).permute(0, 1, 2, 3, 5, 6, 7, 4, 8).reshape(*lead, UNIT, gr, GROUP)
    return ((k * scale[:, :, :, 0]).reshape(*lead[:2], -1, d), (v * scale[:, :, :, 1]).reshape(*lead[:2], -1, d))


def _plain_read(st):
    case, out = st["case"], st["k_out"]
    k, v = _plain_rows(st["cache"], st["read_from"], case["d"])
    live = (st["read_at"][:, None] + torch.arange(case["page"], device=out.device) < st["read_len"][:, None])[:, None, :, None]
    st["k_out"].copy_(torch.where(live, k, torch.zeros_like(k)))
    st["v_out"].copy_(torch.where(live, v, torch.zeros_like(v)))
    return {"k": st["k_out"], "v": st["v_out"]}


def _plain_attend(st):
    case, step = st["case"], st["step"]
    S, d, nkv, window = step.n_seqs, case["d"], case["nkv"], case["window"]
    table = st["table"]
    k, v = _plain_rows(st["cache"], table.clamp(min=0).flatten().long(), d)
    k = k.view(S, -1, *k.shape[1:]).transpose(1, 2).flatten(2, 3)           # [S, nkv, L, d]
    v = v.view(S, -1, *v.shape[1:]).transpose(1, 2).flatten(2, 3)
    seq, place = step.seq_of_token.long(), st["place"]
    G, Q = case["nq"] // nkv, step.max_q_len
    q = torch.zeros(S, Q, nkv, G, d, device=k.device)
    q[seq, place] = st["q"].float().view(-1, nkv, G, d)
    pos = torch.full((S, Q), -1, device=k.device)
    pos[seq, place] = step.positions.long()
    at = torch.arange(k.shape[2], device=k.device)
    first = pos + 1 - window if window > 0 else pos - pos % -window if window < 0 else torch.zeros_like(pos)
    held = (table >= 0).repeat_interleave(case["page"], dim=1)
    seen = (at <= pos[..., None]) & (at >= first[..., None]) & held[:, None]
    x = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.transpose(2, 3)).view(S, nkv, G, Q, -1) * st["scale"]
    x = torch.where(seen[:, None, None], x, torch.full_like(x, float("-inf")))
    sink = st["sink"].view(1, nkv, G, 1, 1) if st["sink"] is not None else torch.full((1, nkv, G, 1, 1), float("-inf"), device=k.device)
    m = torch.maximum(x.amax(-1, keepdim=True), sink)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True) + torch.exp(sink - m)
    o = torch.matmul(p.flatten(2, 3), v).view(S, nkv, G, Q, d) / torch.where(total == 0, torch.ones_like(total), total)
    st["out"].copy_(o.permute(0, 3, 1, 2, 4)[seq, place].flatten(1))
    return st["out"]


# ------------------------------------------------------------------ inputs
def _rows(gen, n, nkv, d, dtype, channels):
    """Keys or values as a projection makes them: some channels of a head much larger than the rest."""
    x = torch.randn(n, nkv, d, generator=gen, device=DEVICE) * channels
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    nkv, d, page = case["nkv"], case["d"], case["page"]
    dtype = getattr(torch, case["dtype"])
    new, kv = _lens(case)
    S, T = len(new), sum(new)
    blocks = [-(-k // page) for k in kv]
    width = max(blocks)
    pool = sum(blocks) + 3
    table = torch.full((S, width), -1, dtype=torch.int32)
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(int(seed))).to(torch.int32)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    table = table.to(DEVICE)
    channels = torch.exp(0.5 * torch.randn(2, nkv, d, generator=gen, device=DEVICE))
    cache = torch.zeros(pool, nkv, page // UNIT, 18 * d, dtype=torch.uint8, device=DEVICE)
    # what the requests have cached: all their rows, or (write) those before the step's
    have = [k - n if case["kind"] == "write" else k for n, k in zip(new, kv)]
    for s, n in enumerate(have):
        for a in range(0, n, 4096):
            p = torch.arange(a, min(n, a + 4096), device=DEVICE)
            rows = [_rows(gen, p.numel(), nkv, d, dtype, c) for c in channels]
            _plain_write(*rows, table[s, p // page].long(), p % page, cache)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    positions = torch.cat([torch.arange(k - n, k) for n, k in zip(new, kv)]).to(torch.int32)
    seq = torch.repeat_interleave(torch.arange(S), torch.tensor(new)).to(torch.int32)
    place = torch.cat([torch.arange(n) for n in new])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    step = SimpleNamespace(
        n_tokens=T, n_seqs=S, positions=positions.to(DEVICE), seq_of_token=seq.to(DEVICE), cu_q=i32(cu), kv_len=i32(kv),
        h_q_start=[k - n for n, k in zip(new, kv)], h_q_len=list(new), h_kv_len=list(kv), max_q_len=max(new), max_kv_len=max(kv),
        decode_only=all(n == 1 for n in new))
    st = dict(case=dict(case), cache=cache, table=table, step=step, place=place.to(DEVICE))
    if case["kind"] == "write":
        # the projection's rows q | k | v side by side, of which the keys and values are views
        proj = torch.randn(T, (case["nq"] + 2 * nkv) * d, generator=gen, device=DEVICE)
        proj[:, case["nq"] * d:] *= channels.reshape(-1)
        proj = proj.to(dtype)
        st["k"] = proj[:, case["nq"] * d:(case["nq"] + nkv) * d].unflatten(1, (nkv, d))
        st["v"] = proj[:, (case["nq"] + nkv) * d:].unflatten(1, (nkv, d))
    if case["kind"] in ("write", "read"):
        # every page that is read back gets the next page of the output
        out_table = torch.full((S, width), -1, dtype=torch.int32)
        pairs = [(s, b) for s in range(S) for b in range(((kv[s] - new[s]) if case["kind"] == "write" else 0) // page, blocks[s])]
        out_table[[s for s, _ in pairs], [b for _, b in pairs]] = torch.arange(len(pairs), dtype=torch.int32)
        st["out_table"] = out_table.to(DEVICE)
        s_of, b_of = (torch.tensor(x, device=DEVICE) for x in zip(*pairs))
        st["read_from"], st["read_at"], st["read_len"] = table[s_of, b_of].long(), b_of * page, step.kv_len[s_of].long()
        st["k_out"], st["v_out"] = (torch.zeros(len(pairs), nkv, page, d, dtype=dtype, device=DEVICE) for _ in range(2))
    if case["kind"] == "write":
        st["page_of"] = table[step.seq_of_token.long(), step.positions.long() // page].long()
    if case["kind"] == "attend":
        st["q"] = (1.5 * torch.randn(T, case["nq"] * d, generator=gen, device=DEVICE)).to(dtype)
        st["out"] = torch.zeros(T, case["nq"] * d, dtype=dtype, device=DEVICE)
        st["scale"] = 1.0 / math.sqrt(d)
        st["sink"] = torch.randn(case["nq"], generator=gen, device=DEVICE) if case["sink"] else None
    return st


def run(state):
    case, step = state["case"], state["step"]
    kind = case["kind"]
    if not own:
        if kind == "attend":
            return _plain_attend(state)
        if kind == "write":
            _plain_write(state["k"], state["v"], state["page_of"], step.positions.long() % case["page"], state["cache"])
        return _plain_read(state)
    from inferloop_b200.csrc import ops
    if kind == "attend":
        ops.kv4_attention(state["q"], state["out"], state["cache"], step, state["table"], case["window"], state["scale"], case["nq"], case["nkv"],
                          case["d"], sink=state["sink"])
        return state["out"]
    if kind == "write":
        ops.kv4_write(state["k"], state["v"], step, state["table"], state["cache"])
    ops.kv4_read(state["cache"], state["table"], step.kv_len, state["out_table"], state["k_out"], state["v_out"])
    return {"k": state["k_out"], "v": state["v_out"]}


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_kept(x):
    """What the cache stands for after it took the rows x, in 64 bits."""
    x = x.double().unflatten(-1, (-1, GROUP))
    s = (x.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).double()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = torch.where(s == 0, torch.zeros_like(x), torch.sign(x) * torch.floor(x.abs() / s + 0.5))
    return (torch.clamp(c, -7, 7) * s).flatten(-2)


def _exact_unit(units, d):
    """Keys and values [n, 16, d] of units [n, 18 d], each element fetched from where the format puts it."""
    dev = units.device
    j, e = torch.arange(UNIT, device=dev)[:, None], torch.arange(d, device=dev)[None]
    g, i = e // 32, e % 32
    byte_k = j * (d // 2) + (i // 8) * (d // 8) + 4 * g + (i % 8) // 2
    byte_v = 8 * d + ((j // 8) * 32 + 4 * (i // 4) + (j // 2) % 4) * (d // 8) + (j % 2) * (d // 16) + 2 * g + (i % 4) // 2
    shift = ((e % 2) * 4).expand(UNIT, d)
    found = []
    for byte, scale0 in ((byte_k, 16 * d), (byte_v, 17 * d)):
        c = ((units[:, byte].int() >> shift) & 15) - 8
        at = scale0 + (j * (d // 32) + g) * 2
        s = (units[:, at].int() << 16 | units[:, at + 1].int() << 24).view(torch.float32)
        found.append(c.double() * s.double())
    return found


def exact(case, seed):
    st = prepare(case, seed)
    d, nkv, page, step = case["d"], case["nkv"], case["page"], st["step"]
    upp = page // UNIT
    rows = {}
    for s in range(step.n_seqs):                           # every request's keys and values [tokens, nkv, d]
        n = step.h_kv_len[s]
        at = st["table"][s, :-(-n // page)].long()
        units = st["cache"][at].transpose(1, 2).reshape(-1, 18 * d)          # [(block, unit, head), bytes]
        k, v = _exact_unit(units, d)
        rows[s] = [x.view(-1, nkv, UNIT, d).transpose(1, 2).reshape(-1, nkv, d)[:n] for x in (k, v)]
        if case["kind"] == "write":
            a, b = int(step.cu_q[s]), int(step.cu_q[s + 1])
            for x, fresh in zip(rows[s], (st["k"], st["v"])):
                x[step.h_q_start[s]:] = _exact_kept(fresh[a:b])
    if case["kind"] != "attend":
        outs = [torch.zeros(x.shape, dtype=F64, device=DEVICE) for x in (st["k_out"], st["v_out"])]
        goes = st["out_table"].tolist()
        for s in range(step.n_seqs):
            for b, to in enumerate(goes[s]):
                if to >= 0:
                    for x, o in zip(rows[s], outs):
                        part = x[b * page:(b + 1) * page]
                        o[to, :, :part.shape[0]] = part.transpose(0, 1)
        return {"k": outs[0], "v": outs[1]}
    G = case["nq"] // nkv
    out = torch.zeros(st["out"].shape, dtype=F64, device=DEVICE)
    for s in range(step.n_seqs):
        a, n = int(step.cu_q[s]), step.h_q_len[s]
        k, v = rows[s]
        pos = torch.arange(step.h_q_start[s], step.h_kv_len[s], device=DEVICE)
        key = torch.arange(k.shape[0], device=DEVICE)
        lo = torch.tensor([_first_key(p, case["window"]) for p in range(step.h_q_start[s], step.h_kv_len[s])], device=DEVICE)
        seen = (key[None] <= pos[:, None]) & (key[None] >= lo[:, None])
        for h in range(case["nq"]):
            x = st["q"][a:a + n, h * d:(h + 1) * d].double() @ k[:, h // G].t() * st["scale"]
            x = x.masked_fill(~seen, float("-inf"))
            if st["sink"] is not None:
                x = torch.cat([x, st["sink"][h].double().expand(n, 1)], dim=1)
            p = torch.softmax(x, dim=1)[:, :k.shape[0]]
            out[a:a + n, h * d:(h + 1) * d] = p @ v[:, h // G]
    return out
