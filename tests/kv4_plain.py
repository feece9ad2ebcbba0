"""The 4-bit key/value cache stated plainly, in 64 bits: what rows become, where every code lies, attention over what is held."""
from types import SimpleNamespace

import torch

GROUP, UNIT = 32, 16


def kept(x):
    """(codes, scales, values) that rows [..., d] of x are kept as."""
    g = x.double().unflatten(-1, (-1, GROUP))
    s = (g.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).double()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    c = torch.where((s == 0) | bad, torch.zeros_like(g), torch.sign(g) * torch.floor(g.abs() / torch.where(s == 0, torch.ones_like(s), s) + 0.5))
    c = c.clamp(-7, 7)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    return c.flatten(-2), s.squeeze(-1), (c * s).flatten(-2)


def places(d):
    """Byte and shift of every code of a unit, (keys, values) as [16, d] each, and the bytes of the scales [2, 16, d / 32]."""
    key, value, shift = (torch.zeros(UNIT, d, dtype=torch.long) for _ in range(3))
    for j in range(UNIT):
        for e in range(d):
            g, i = divmod(e, 32)
            key[j, e] = j * (d // 2) + (i // 8) * (d // 8) + 4 * g + (i % 8) // 2
            value[j, e] = 8 * d + ((j // 8) * 32 + 4 * (i // 4) + (j // 2) % 4) * (d // 8) + (j % 2) * (d // 16) + 2 * g + (i % 4) // 2
            shift[j, e] = 4 * (e % 2)
    scale = torch.arange(2 * UNIT * (d // 32)).view(2, UNIT, d // 32) * 2 + 16 * d
    return key, value, shift, scale


def write(cache, pages, slots, k, v):
    """Rows k, v [T, nkv, d] into the cache (a uint8 tensor on the CPU) at (page, slot) each."""
    d = k.shape[-1]
    key, value, shift, scale = places(d)
    pages, slots, heads = torch.as_tensor(pages).long(), torch.as_tensor(slots).long(), torch.arange(k.shape[1])
    j = slots % UNIT
    unit = (pages[:, None, None], heads[None, :, None], (slots // UNIT)[:, None, None])
    for x, place, which in ((k, key, 0), (v, value, 1)):
        c, s, _ = kept(x)
        c, s = (c + 8).to(torch.uint8), s.to(torch.bfloat16).view(torch.int16).int() & 0xffff
        cache[(*unit, place[j, ::2][:, None])] = c[..., ::2] | c[..., 1::2] << 4          # (a byte holds two elements of one row)
        cache[(*unit, scale[which, j][:, None])] = (s & 255).to(torch.uint8)
        cache[(*unit, scale[which, j][:, None] + 1)] = (s >> 8).to(torch.uint8)


def rows(cache, pages):
    """(keys, values) [n, nkv, page_size, d] that the pages stand for."""
    d = cache.shape[-1] // 18
    units = cache[pages].cpu()
    key, value, shift, scale = places(d)
    found = []
    for place, at in ((key, scale[0]), (value, scale[1])):
        c = ((units[..., place].int() >> shift) & 15) - 8
        s = ((units[..., at].int() | units[..., at + 1].int() << 8) << 16).view(torch.float32).double()
        x = (c.double().unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)
        found.append(x.flatten(2, 3))
    return found


def first_key(pos, window):
    return max(0, pos + 1 - window) if window > 0 else pos - pos % -window if window < 0 else 0


def attention(q, cache, table, starts, lens, window, scale, nq, nkv, sink=None):
    """q [T, nq * d] of sequences that bring lens[s] tokens from position starts[s] on -> ([T, nq * d] in 64 bits, largest score)."""
    d = q.shape[1] // nq
    page = cache.shape[2] * UNIT
    out, t, most = torch.zeros(q.shape, dtype=torch.float64), 0, 0.0
    q, table = q.double().cpu(), table.cpu()
    for s, n in enumerate(lens):
        if n == 0:
            continue
        blocks = -(-(starts[s] + n) // page)
        k, v = (x.transpose(1, 2).flatten(0, 1) for x in rows(cache, table[s, :blocks].clamp(min=0).long()))
        held = (table[s, :blocks] >= 0).repeat_interleave(page)
        for i in range(n):
            pos = starts[s] + i
            at = torch.arange(first_key(pos, window), pos + 1)
            at = at[held[at]]
            for h in range(nq):
                x = k[at, h // (nq // nkv)] @ q[t, h * d:(h + 1) * d] * scale
                if sink is not None:
                    x = torch.cat([x, sink[h:h + 1].double().cpu()])
                if x.numel() == 0:
                    continue
                most = max(most, float(x.abs().max()))
                p = torch.softmax(x, 0)[:at.numel()]
                out[t, h * d:(h + 1) * d] = p @ v[at, h // (nq // nkv)]
            t += 1
    return out, most


def make_step(starts, lens, device):
    """The step that brings lens[s] tokens of sequence s from position starts[s] on."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    kv = [a + n for a, n in zip(starts, lens)]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return SimpleNamespace(
        n_tokens=cu[-1], n_seqs=len(lens), positions=i32([a + i for a, n in zip(starts, lens) for i in range(n)]),
        seq_of_token=i32([s for s, n in enumerate(lens) for _ in range(n)]), cu_q=i32(cu), kv_len=i32(kv), h_q_start=list(starts), h_q_len=list(lens),
        h_kv_len=kv, max_q_len=max(lens), max_kv_len=max(kv), decode_only=all(n == 1 for n in lens))


def make_table(kv, page, spare, seed):
    """Block table [S, max blocks] with pages in random order, and the pool's size."""
    blocks = [-(-n // page) for n in kv]
    pool = sum(blocks) + spare
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(kv), max(1, max(blocks))), -1, dtype=torch.int32)
    for s, b in enumerate(blocks):
        for i in range(b):
            table[s, i] = order.pop()
    return table, pool
