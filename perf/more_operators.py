"""Beam search: selection over beams and vocabulary, reordering of the cache, steps laid out on the device, attention of beams that
share pages, as cases that can be timed and checked.

A request has W beams, rows r W .. r W + W - 1 of a step.  Each row has a block table of its own; full pages are shared by the beams that
descend from the same tokens (a prompt's by all of them), the last, partly filled page of a row is its own.

The kinds of pass:

  select   the k best continuations (beam, token) of every request by score + log softmax(logits), best first
  reorder  beams continue their parents: block tables follow them, the parent's last page and its state are copied for every child but the first
  build    from the tokens that each sequence has and brings: positions, offsets, lengths, slot map, and new pages in the block tables
  attend   one new token of every beam attends to all that its row has in the cache

Sizes are those of bench.py and of the tests: a vocabulary of 151,936, 32 / 8, 40 / 8 and 64 / 8 heads of 128, pages of 16 tokens, and small
models with heads of 64 and 32.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
F64 = torch.float64
NEG = float("-inf")


def _select(name, requests, beams, k, vocab=151936, dtype="float32", first=False, masked=False):
    """first: the step after the prompt, when only the first beam is alive; masked: some tokens are forbidden (logits of -inf)."""
    c = dict(kind="select", requests=requests, beams=beams, k=k, vocab=vocab, dtype=dtype, first=first, masked=masked)
    return dict(c, name=name) if name else c


def _reorder(name, requests, beams, prompt, made, layers=36, nkv=8, d=128, page=16, dtype="bfloat16", bits=16, pool=0, slots=0):
    """made: tokens that every beam has generated; bits 4: the packed cache; pool: a second set of pages with a row for so many tokens;
    slots: floats of recurrent state that a layer keeps for a request (0: none)."""
    c = dict(kind="reorder", requests=requests, beams=beams, prompt=prompt, made=made, layers=layers, nkv=nkv, d=d, page=page, dtype=dtype, bits=bits,
             pool=pool, slots=slots)
    return dict(c, name=name) if name else c


def _build(name, sequences, tokens, cached, page=16, pool=0):
    """tokens: what the sequence that brings the most brings (1: a decode step); cached: what the longest has."""
    c = dict(kind="build", sequences=sequences, tokens=tokens, cached=cached, page=page, pool=pool)
    return dict(c, name=name) if name else c


def _attend(name, requests, beams, prompt, made, nq=32, nkv=8, d=128, page=16, dtype="bfloat16", window=0, sink=False):
    """window: keys that a token sees (0: all; negative: those of its aligned chunk); sink: a logit a head in the denominator."""
    c = dict(kind="attend", requests=requests, beams=beams, prompt=prompt, made=made, nq=nq, nkv=nkv, d=d, page=page, dtype=dtype, window=window, sink=sink)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's search with four beams: a launch's latency over two and a half megabytes of logits
        _select("select 1 x 4", 1, 4, 8),
        # an odd batch of small models, five beams and three candidates a beam, forbidden tokens
        _select("select 7 x 5 of 32003", 7, 5, 15, vocab=32003, masked=True),
        # the largest batch that one step takes: 64 requests of four beams
        _select("select 64 x 4", 64, 4, 8),
        # one user: 36 layers' last pages and nothing else moves
        _reorder("reorder 1 x 4", 1, 4, 1024, 41),
        # a full batch of eight beams behind prompts of 1,024 tokens, 40 layers
        _reorder("reorder 8 x 8", 8, 8, 1024, 27, layers=40),
        # recurrent layers: the state of 512 KB a layer and request follows the beams, beside few attention layers
        _reorder("reorder 6 x 5 with state", 6, 5, 300, 75, layers=4, nkv=2, d=64, slots=131072),
        # a decode step of 64 requests of four beams
        _build("build 256 tokens", 256, 1, 1200),
        # portions of prompts beside decoding sequences, the largest step of a server
        _build("build 33 sequences, portions of 2048", 33, 2048, 5000),
        # one user's search: latency
        _attend("attend 1 x 4 x 1030", 1, 4, 1000, 30),
        # a busy server: 16 requests of four beams
        _attend("attend 16 x 4 x 1100", 16, 4, 1030, 70),
        # long documents, eight beams, 40 / 8 heads
        _attend("attend 6 x 8 x 6000", 6, 8, 5940, 61, nq=40),
        # the 32-bit engine, a window, a learned sink, small heads
        _attend("attend float32 3 x 4 x 700", 3, 4, 650, 51, nq=8, nkv=2, d=64, dtype="float32", window=500, sink=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["select", "select", "reorder", "build", "attend", "attend", "attend"])
    beams = rng.choice([1, 2, 3, 4, 4, 5, 6, 8, 8, 12, 16])
    if kind == "select":
        vocab = _log(rng, 300, 151936)
        requests = _log(rng, 1, max(1, min(256 // beams, 32000000 // (vocab * beams))))
        return _select(None, requests, beams, min(64, beams * rng.choice([1, 2, 2, 3])), vocab, rng.choice(["float32", "float32", "bfloat16"]),
                       rng.random() < 0.15, rng.random() < 0.3)
    if kind == "build":
        if rng.random() < 0.5:
            return _build(None, _log(rng, 1, 256), 1, _log(rng, 1, 9000) - 1, rng.choice([16, 16, 32, 64]), rng.choice([0, 0, 16]))
        n = _log(rng, 1, 64)
        return _build(None, n, _log(rng, 2, 2048), _log(rng, 1, 9000) - 1, rng.choice([16, 16, 32, 64]), rng.choice([0, 0, 16]))
    nkv = rng.choice([1, 2, 4, 8, 8, 8])
    d = rng.choice([32, 64, 64, 96, 128, 128, 128])
    page = rng.choice([16, 16, 16, 32, 64, 128])
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    made = _log(rng, 1, 200) - 1
    if kind == "reorder":
        requests = _log(rng, 1, max(1, 64 // beams))
        bits = 4 if rng.random() < 0.25 else 16
        pool = 16 if bits == 16 and rng.random() < 0.2 else 0
        slots = _log(rng, 64, 20000) if rng.random() < 0.3 else 0
        return _reorder(None, requests, beams, _log(rng, 1, 1200), made, rng.randint(1, 24), nkv, d, page, dtype, bits, pool, slots)
    group = rng.choice([1, 2, 3, 4, 4, 4, 5, 8, 8])
    window = rng.choice([0, 0, 0, 0, 40, 500, -256])
    requests = _log(rng, 1, max(1, 64 // beams))
    prompt = _log(rng, 1, max(1, min(20000, 40000 // requests)))
    if dtype == "float32":
        prompt, group = min(prompt, 2000), min(group, 4)
    return _attend(None, requests, beams, prompt, made, nkv * group, nkv, d, page, dtype, window, rng.random() < 0.2)


# ------------------------------------------------------------------ what the requests have
def _lens(case):
    """(prompt, tokens in the cache) of each request: ragged prompts, the first the longest."""
    prompts = [max(1, case["prompt"] - (r * 41) % (case["prompt"] // 4 + 1)) for r in range(case["requests"])]
    return prompts, [p + case["made"] for p in prompts]


def _owners(case, r, rows_prompt, rows, last_own):
    """[W][blocks]: whose page each beam's block is (-1: the prompt's, shared).  From block to block the beams pick parents anew, so that
    early blocks are shared by most.  last_own: the last block, partly filled or the newest, is every beam's own."""
    W, page = case["beams"], case["page"]
    rng = random.Random(9176 * r + W)
    blocks = -(-rows // page)
    found = [[-1] * blocks for _ in range(W)]
    line = list(range(W))
    for b in reversed(range(rows_prompt // page, blocks)):
        if b < blocks - 1 or not last_own:
            parent = [min(int(W * rng.random() ** 1.5), W - 1) for _ in range(W)]
            line = [parent[x] for x in line]
        for w in range(W):
            found[w][b] = line[w]
    return found


def _tables(case, order, stride=1):
    """Block tables [R W, widest] (int32, host), the pages of the pool and one that is not held; order(n): a shuffled pool of n."""
    prompts, lens = _lens(case)
    page, W = case["page"], case["beams"]
    rows, pairs, ids = [], [], {}
    for r, (p, n) in enumerate(zip(prompts, lens)):
        have = n // stride
        for w, line in enumerate(_owners(case, r, p // stride, have, have % page != 0 or stride > 1)):
            rows.append([(r, b, o) for b, o in enumerate(line)])
    for line in rows:
        for key in line:
            if key not in ids:
                ids[key] = len(ids)
    shuffled = order(len(ids) + 3)
    width = max(1, max(len(x) for x in rows) + 1)
    table = torch.full((len(rows), width), -1, dtype=torch.int32)
    for i, line in enumerate(rows):
        if line:
            table[i, :len(line)] = torch.tensor([int(shuffled[ids[key]]) for key in line], dtype=torch.int32)
    return table, len(ids) + 3, int(shuffled[len(ids)])


def _first_key(pos, window):
    return max(0, pos + 1 - window) if window > 0 else pos - pos % -window if window < 0 else 0


def _brought(case):
    """(tokens brought, tokens cached before) of each sequence of a step."""
    n = case["sequences"]
    new = [1 if case["tokens"] == 1 or s % 3 == 2 else max(1, case["tokens"] - (s * 331) % case["tokens"]) for s in range(n)]
    return new, [max(0, case["cached"] - (s * 37) % (case["cached"] + 1)) for s in range(n)]


def _strides(case):
    return [1] + ([case["pool"]] if case["pool"] else [])


def work(case):
    kind = case["kind"]
    if kind == "select":
        n = case["requests"] * case["beams"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "float32" else 2) + case["requests"] * (case["beams"] * 8 + case["k"] * 12), "flops": 4 * n}
    if kind == "build":
        new, cached = _brought(case)
        total = sum(new) * 16 + case["sequences"] * 16
        for s in _strides(case):
            total += 8 * sum(-(-((c + n) // s) // case["page"]) - -(-(c // s) // case["page"]) for n, c in zip(new, cached))
        return {"bytes": total, "flops": 0}
    e = 4 if case["dtype"] == "float32" else 2
    W, page, nkv, d = case["beams"], case["page"], case["nkv"], case["d"]
    prompts, lens = _lens(case)
    if kind == "reorder":
        # a third of the children are not their parent's first
        copies = case["requests"] * max(1, W // 3) if W > 1 else 0
        row = case["layers"] * nkv * d
        total = 0
        for s in _strides(case):
            fill = sum(n // s % page for n in lens) / len(lens)
            total += int(copies * fill) * 2 * row * (2 * e if case["bits"] == 16 else 9 / 8)
            total += sum(W * -(-(n // s) // page) * 8 for n in lens)
        return {"bytes": int(total) + copies * 2 * case["layers"] * case["slots"] * 4 + case["requests"] * W * 20, "flops": 0}
    keys = pairs = 0
    for r, (p, n) in enumerate(zip(prompts, lens)):
        first = _first_key(n - 1, case["window"])
        pairs += W * (n - first)
        own = _owners(case, r, p, n, n % page != 0)
        for b in range(first // page, -(-n // page)):
            keys += len({own[w][b] for w in range(W)}) * (min(n, (b + 1) * page) - max(first, b * page))
    rows = case["requests"] * W
    return {"bytes": keys * 2 * nkv * d * e + 2 * rows * case["nq"] * d * e, "flops": 4 * pairs * case["nq"] * d}


# ------------------------------------------------------------------ the plain form
def _plain_select(st):
    case = st["case"]
    R, W, k = case["requests"], case["beams"], case["k"]
    x = st["logits"].float()
    bad = (torch.isnan(x) | (x == float("inf"))).any(1)
    top = torch.where(bad[:, None], torch.full_like(x, NEG), x)
    m = top.amax(1, keepdim=True).double()
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    lse = m + torch.log(torch.exp(top.double() - m).sum(1, keepdim=True))
    best, token = torch.sort(top, dim=1, descending=True, stable=True)
    best, token = best[:, :k], token[:, :k]
    base = st["scores"].view(-1, 1).double() - lse
    s = torch.where(torch.isinf(best) | torch.isnan(base) | torch.isinf(base), torch.full_like(base, NEG), base + best.double())
    n = best.shape[1]
    s, best, token = s.view(R, -1), best.reshape(R, -1), token.reshape(R, -1)
    beam = (torch.arange(W * n, device=s.device) // n).expand(R, -1)
    at = torch.sort(best, dim=1, descending=True, stable=True).indices
    at = at.gather(1, torch.sort(s.gather(1, at), dim=1, descending=True, stable=True).indices)[:, :k]
    s, token, beam = (t.gather(1, at) for t in (s, token, beam))
    none = torch.isinf(s)
    out = {"scores": st["out_scores"].fill_(NEG), "parents": st["parents"].fill_(-1), "tokens": st["tokens"].fill_(-1), "bad": st["bad"].copy_(bad)}
    out["scores"][:, :s.shape[1]] = s.float()
    out["parents"][:, :s.shape[1]] = torch.where(none, torch.full_like(beam, -1), beam).int()
    out["tokens"][:, :s.shape[1]] = torch.where(none, torch.full_like(token, -1), token).int()
    return out


def _plain_places(parents):
    """Whose place (last page and slot) every child takes [R, W], and where its rows are copied from (-1: it takes its parent's place)."""
    R, W = parents.shape
    child = torch.arange(W, device=parents.device)
    p = parents.long()
    same = (p[:, :, None] == p[:, None, :]) & (p >= 0)[:, :, None] & (child[None, :] < child[:, None])
    first = (p >= 0) & ~same.any(2)
    taken = ((p[:, :, None] == child) & first[:, :, None]).any(1)
    free_at = torch.sort(taken.long(), dim=1, stable=True).indices        # the places nobody takes over, in order
    turn = torch.cumsum((~first).long(), 1) - 1
    place = torch.where(first, p, free_at.gather(1, turn.clamp(min=0)))
    return place, torch.where(first | (p < 0), torch.full_like(p, -1), p)


def _plain_reorder(st):
    case = st["case"]
    R, W, page = case["requests"], case["beams"], case["page"]
    place, source = _plain_places(st["parents"])
    first_row = (torch.arange(R, device=place.device) * W)[:, None]
    follow = (torch.where(st["parents"] >= 0, st["parents"].long(), torch.arange(W, device=place.device).expand(R, W)) + first_row).flatten()
    places, copied = (place + first_row).flatten(), source.flatten() >= 0
    sources = (source.clamp(min=0) + first_row).flatten()
    for (table, storages, stride), spare in zip(st["groups"], st["spare"]):
        rows = st["kv_len"].long() // stride
        fill, last = rows % page, (rows // page).clamp(max=table.shape[1] - 1)
        held = table.gather(1, last[:, None])[:, 0]
        # rows that copy nothing write a page that nobody holds over itself
        moves = copied & (fill > 0)
        a, b = (torch.where(moves, held[i].long(), torch.full_like(i, spare)) for i in (sources, places))
        for x in storages:
            if case["bits"] == 4:
                live = torch.arange(x.shape[3], device=x.device) < torch.div(fill + 15, 16, rounding_mode="floor")[:, None]
                x[:, b] = torch.where(live[:, None, :, None], x[:, a], x[:, b])
            else:
                live = torch.arange(page, device=x.device) < fill[:, None]
                x[:, :, b] = torch.where(live[:, None, :, None], x[:, :, a], x[:, :, b])
        fresh = table[follow]
        fresh.scatter_(1, last[:, None], torch.where((fill > 0)[:, None], held[places][:, None], fresh.gather(1, last[:, None])))
        # (entries behind the rows in use stay as they are)
        used = torch.arange(table.shape[1], device=table.device) < torch.div(rows + page - 1, page, rounding_mode="floor")[:, None]
        table.copy_(torch.where(used, fresh, table))
    slots = st["slots"].long()
    taken = slots[places]
    for x in st["states"]:
        x[taken] = x[torch.where(copied, slots[sources], taken)]
    st["slots"].copy_(taken.int())
    return _moved(st)


def _moved(st):
    return {"tables": [t for t, _, _ in st["groups"]], "pages": [x for _, xs, _ in st["groups"] for x in xs], "slots": st["slots"], "states": st["states"]}


def _plain_build(st):
    case, page = st["case"], st["case"]["page"]
    new, cached = st["new"].long(), st["cached"].long()
    after = cached + new
    ends = torch.cumsum(new, 0)
    st["cu_q"][0] = 0
    st["cu_q"][1:] = ends.int()
    st["kv_len"].copy_(after)
    T = st["positions"].numel()
    at = torch.arange(T, device=new.device)
    seq = torch.searchsorted(ends, at, right=True)
    st["seq_of_token"].copy_(seq)
    pos = cached[seq] + at - (ends - new)[seq]
    st["positions"].copy_(pos)
    for g in st["pages"]:
        had = torch.div(torch.div(cached, g.stride, rounding_mode="floor") + page - 1, page, rounding_mode="floor")
        want = torch.div(torch.div(after, g.stride, rounding_mode="floor") + page - 1, page, rounding_mode="floor")
        need = want - had
        before = torch.cumsum(need, 0) - need + g.used.long()
        b = torch.arange(g.table.shape[1], device=new.device)
        fresh = (b >= had[:, None]) & (b < want[:, None])
        ids = g.free[(before[:, None] + b - had[:, None]).clamp(0, g.free.numel() - 1)]
        g.table.copy_(torch.where(fresh, ids, g.table))
        g.used_out.copy_(g.used + need.sum())
    held = st["pages"][0].table[seq, torch.div(pos, page, rounding_mode="floor")].long()
    st["slot_map"].copy_(torch.where(held >= 0, held * page + pos % page, torch.full_like(held, -1)))
    return _laid_out(st)


def _laid_out(st):
    return {"positions": st["positions"], "seq_of_token": st["seq_of_token"], "cu_q": st["cu_q"], "kv_len": st["kv_len"], "slot_map": st["slot_map"],
            "tables": [g.table for g in st["pages"]], "used": [g.used_out for g in st["pages"]]}


def _plain_attend(st):
    case = st["case"]
    W, d, nkv, window, page = case["beams"], case["d"], case["nkv"], case["window"], case["page"]
    G = case["nq"] // nkv
    table, pos = st["table"], st["step"].positions.long()
    at = torch.arange(table.shape[1] * page, device=table.device)
    for r in range(case["requests"]):
        own_rows = slice(r * W, r * W + W)
        ids, where = table[own_rows], pos[own_rows]
        k, v = (c[ids.clamp(min=0).long()].transpose(1, 2).flatten(2, 3).float() for c in (st["k_cache"], st["v_cache"]))       # [W, nkv, L, d]
        first = where + 1 - window if window > 0 else where - where % -window if window < 0 else torch.zeros_like(where)
        seen = (at <= where[:, None]) & (at >= first[:, None]) & (ids >= 0).repeat_interleave(page, dim=1)
        x = torch.matmul(st["q"][own_rows].float().view(W, nkv, G, d), k.transpose(2, 3)) * st["scale"]
        x = torch.where(seen[:, None, None], x, torch.full_like(x, NEG))
        v = torch.where(seen[:, None, :, None], v, torch.zeros_like(v))
        sink = st["sink"].view(1, nkv, G, 1) if st["sink"] is not None else torch.full((1, nkv, G, 1), NEG, device=k.device)
        m = torch.maximum(x.amax(-1, keepdim=True), sink)
        m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
        p = torch.exp(x - m)
        total = p.sum(-1, keepdim=True) + torch.exp(sink - m)
        o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
        st["out"][own_rows] = o.flatten(1).to(st["out"].dtype)
    return st["out"]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    host = np.random.default_rng(int(seed))
    kind = case["kind"]
    st = dict(case=dict(case))
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(DEVICE)  # noqa: E731
    if kind == "select":
        R, W, V, k = case["requests"], case["beams"], case["vocab"], case["k"]
        # a few tokens stand out, as behind a trained model's output matrix
        x = 2.5 * torch.randn(R * W, V, generator=gen, device=DEVICE)
        peaks = torch.randint(0, V, (R * W, 12), generator=gen, device=DEVICE)
        x.scatter_add_(1, peaks, 6 * torch.rand(R * W, 12, generator=gen, device=DEVICE))
        if case["masked"]:
            x[:, ::7] = NEG
        scores = -40 * torch.rand(R, W, generator=gen, device=DEVICE)
        scores, _ = torch.sort(scores, dim=1, descending=True)
        if case["first"]:
            scores[:, 0], scores[:, 1:] = 0, NEG
        return dict(st, logits=x.to(getattr(torch, case["dtype"])), scores=scores, parents=torch.zeros(R, k, dtype=torch.int32, device=DEVICE),
                    tokens=torch.zeros(R, k, dtype=torch.int32, device=DEVICE), out_scores=torch.zeros(R, k, device=DEVICE),
                    bad=torch.zeros(R * W, dtype=torch.int32, device=DEVICE))
    if kind == "build":
        new, cached = _brought(case)
        page, pages = case["page"], []
        for stride in _strides(case):
            had = [-(-(c // stride) // page) for c in cached]
            want = [-(-((c + n) // stride) // page) for n, c in zip(new, cached)]
            pool = host.permutation(sum(want) + 17).astype(np.int32)
            table = np.full((len(new), max(max(want), 1) + 2), -1, dtype=np.int32)
            used = 0
            for s, n in enumerate(had):
                table[s, :n] = pool[used:used + n]
                used += n
            pages.append(SimpleNamespace(table=i32(table), free=i32(pool), used=i32([used]), used_out=i32([0]), page_size=page, stride=stride))
        T, S = sum(new), len(new)
        zeros = lambda n, dtype=torch.int32: torch.zeros(n, dtype=dtype, device=DEVICE)  # noqa: E731
        return dict(st, new=i32(new), cached=i32(cached), positions=zeros(T), seq_of_token=zeros(T), cu_q=zeros(S + 1), kv_len=zeros(S),
                    slot_map=zeros(T, torch.int64), pages=pages, refused=zeros(1))
    _, lens = _lens(case)
    W, nkv, d, page = case["beams"], case["nkv"], case["d"], case["page"]
    dtype = getattr(torch, case["dtype"])
    kv_len = i32([n for n in lens for _ in range(W)])
    if kind == "attend":
        table, pool, _ = _tables(case, host.permutation)
        channels = torch.exp(0.5 * torch.randn(2, nkv, 1, d, generator=gen, device=DEVICE))
        k, v = ((torch.randn(pool, nkv, page, d, generator=gen, device=DEVICE) * c).to(dtype) for c in channels)
        step = SimpleNamespace(n_tokens=kv_len.numel(), n_seqs=kv_len.numel(), positions=kv_len - 1, kv_len=kv_len,
                               cu_q=i32(list(range(kv_len.numel() + 1))), seq_of_token=i32(list(range(kv_len.numel()))),
                               max_kv_len=max(lens), decode_only=True)
        q = (1.5 * torch.randn(kv_len.numel(), case["nq"] * d, generator=gen, device=DEVICE)).to(dtype)
        return dict(st, table=table.to(DEVICE), k_cache=k, v_cache=v, step=step, q=q, out=torch.zeros_like(q), scale=1.0 / math.sqrt(d),
                    sink=torch.randn(case["nq"], generator=gen, device=DEVICE) if case["sink"] else None)
    groups, spare = [], []
    for stride in _strides(case):
        table, pool, unheld = _tables(case, host.permutation, stride)
        spare.append(unheld)
        if case["bits"] == 4:
            x = torch.randint(0, 256, (case["layers"], pool, nkv, page // 16, 18 * d), generator=gen, device=DEVICE, dtype=torch.uint8)
        else:
            x = torch.randn(case["layers"], 2, pool, nkv, page, d, generator=gen, device=DEVICE, dtype=dtype)
        groups.append((table.to(DEVICE), [x], stride))
    R = case["requests"]
    parents = np.minimum((W * host.random((R, W)) ** 1.5).astype(np.int32), W - 1)
    slots = host.permutation(R * W + 2)[:R * W]
    states = [torch.randn(R * W + 2, case["slots"], generator=gen, device=DEVICE) for _ in range(case["layers"])] if case["slots"] else []
    st.update(groups=groups, spare=spare, parents=i32(parents), slots=i32(slots), states=states, kv_len=kv_len)
    if own:
        # the storage that beams move in, described once beside the cache
        from inferloop_b200.csrc import ops
        st["handle"] = ops.BeamState([(xs, page, stride) for _, xs, stride in groups], states, DEVICE)
    return st


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"select": _plain_select, "reorder": _plain_reorder, "build": _plain_build, "attend": _plain_attend}[kind](state)
    from inferloop_b200.csrc import ops
    case = state["case"]
    if kind == "select":
        ops.beam_select(state["logits"], state["scores"], state["parents"], state["tokens"], state["out_scores"], state["bad"])
        return {"scores": state["out_scores"], "parents": state["parents"], "tokens": state["tokens"], "bad": state["bad"]}
    if kind == "reorder":
        ops.beam_reorder(state["handle"], state["parents"], state["kv_len"], [t for t, _, _ in state["groups"]], state["slots"])
        return _moved(state)
    if kind == "build":
        ops.step_build(state["new"], state["cached"], state["kv_len"], state["positions"], state["seq_of_token"], state["cu_q"],
                       [ops.StepPages(g.table, g.free, g.used, g.page_size, g.stride, g.used_out) for g in state["pages"]], state["refused"],
                       slot_map=state["slot_map"])
        return _laid_out(state)
    ops.attention_beams(state["q"], state["out"], state["k_cache"], state["v_cache"], state["step"], state["table"], case["beams"], case["window"],
                        state["scale"], case["nq"], case["nkv"], case["d"], sink=state["sink"])
    return state["out"]


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_select(st):
    case = st["case"]
    R, W, V, k = case["requests"], case["beams"], case["vocab"], case["k"]
    out = {"scores": torch.full((R, k), NEG, dtype=F64), "parents": torch.full((R, k), -1, dtype=torch.int32),
           "tokens": torch.full((R, k), -1, dtype=torch.int32), "bad": torch.zeros(R * W, dtype=torch.int32)}
    for r in range(R):
        x = st["logits"][r * W:(r + 1) * W].double()
        s = torch.log_softmax(x, dim=1) + st["scores"][r].double()[:, None]
        s, x = s.flatten(), x.flatten()
        s = torch.where(torch.isnan(s), torch.full_like(s, NEG), s)
        border = torch.topk(s, min(k, s.numel())).values[-1]
        at = torch.nonzero((s >= border - 1e-9) & (s > NEG)).flatten().cpu().numpy()
        a, b = s.cpu().numpy()[at], x.cpu().numpy()[at]
        at = at[np.lexsort((at, -b, -a))][:k]
        out["scores"][r, :len(at)] = s.cpu()[torch.from_numpy(at)]
        out["parents"][r, :len(at)] = torch.from_numpy(at // V).int()
        out["tokens"][r, :len(at)] = torch.from_numpy(at % V).int()
    return out


def _exact_attend(st):
    case, step = st["case"], st["step"]
    d, nkv, page, W = case["d"], case["nkv"], case["page"], case["beams"]
    G = case["nq"] // nkv
    out = torch.zeros(st["out"].shape, dtype=F64, device=DEVICE)
    table, pos = st["table"].cpu(), step.positions.tolist()
    for i, p in enumerate(pos):
        lo = _first_key(p, case["window"])
        key = torch.arange(lo, p + 1)
        at = table[i, key // page].long().to(DEVICE)
        k, v = (c[at, :, (key % page).to(DEVICE)].double() for c in (st["k_cache"], st["v_cache"]))         # [keys, nkv, d]
        q = st["q"][i].double().view(nkv, G, d)
        x = torch.einsum("hgd,nhd->hgn", q, k) * st["scale"]
        if st["sink"] is not None:
            x = torch.cat([x, st["sink"].double().view(nkv, G, 1)], dim=2)
        out[i] = torch.einsum("hgn,nhd->hgd", torch.softmax(x, dim=2)[..., :len(key)], v).flatten()
    return out


def exact(case, seed):
    if case["kind"] not in ("select", "attend"):
        return None                                    # whole numbers and moved bytes: nothing is computed
    st = prepare(case, seed)
    return _exact_select(st) if case["kind"] == "select" else _exact_attend(st)
