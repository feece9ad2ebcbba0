"""Attention over the 4-bit cache from bfloat16 queries: the result in 64 bits and how far from it the kernels may be, element by element.

With p the probabilities that a token gives its keys, v their values:

  2^-8 |result|        the result is rounded to bfloat16 (2^-9), and once more for what lies between
  2^-10 sum p |v|      probabilities times scale, or probabilities, are rounded to fp16 (2^-11 each)
  2 d sum p |v|        a score that is off by d moves its weight by a factor exp(d).  The operands of a group of 32 elements carry offsets of
                       up to 1032 that are taken out again: their 32-bit sum is off by some 8 roundings of 2^-23 of (1032 + 7) s |q|, which is
                       d = 8 x 2^-23 x 1039 / 7 x (the group's largest key times |q|, summed over the groups) = 2^-9.7 / 7 of it
  floor                where fp16 has no normal numbers left, a factor is off by 2^-25.  Rows: p times scale, whose unit takes in 2^6 over the largest
                       p and the largest scale.  Unpacked tiles: p, whose unit takes in 2^7 over the largest p times its tile's (of 128 keys)
                       largest value.  A factor 2 on either, values being 7 scales but for a rounding and scales a power of two but for 2.
"""
import torch

import kv4_plain as plain

TILE = 128


def outcome(q, cache, table, starts, lens, window, scale, nq, nkv, sink=None, unpacked=False):
    """(result, bound), [T, nq * d] in 64 bits each, of queries q [T, nq * d] of sequences that bring lens[s] tokens from position starts[s] on."""
    d, page, G = q.shape[1] // nq, cache.shape[2] * plain.UNIT, nq // nkv
    q, table = q.double().cpu(), table.cpu()
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    t = 0
    for s, n in enumerate(lens):
        if n == 0:
            continue
        blocks = -(-(starts[s] + n) // page)
        k, v = (x.transpose(1, 2).flatten(0, 1) for x in plain.rows(cache, table[s, :blocks].clamp(min=0).long()))      # [L, nkv, d]
        L = k.shape[0]
        at, pos = torch.arange(L), torch.arange(starts[s], starts[s] + n)
        first = torch.tensor([plain.first_key(int(p), window) for p in pos])
        seen = (at <= pos[:, None]) & (at >= first[:, None]) & (table[s, :blocks] >= 0).repeat_interleave(page)
        any_seen = seen.any(0)
        for h in range(nq):
            kh, vh = k[:, h // G], torch.where(any_seen[:, None], v[:, h // G], 0.0)
            qh = q[t:t + n, h * d:(h + 1) * d]
            x = (qh @ kh.T * scale).masked_fill(~seen, float("-inf"))
            if sink is not None:
                x = torch.cat([x, sink[h:h + 1].double().cpu().expand(n, 1)], dim=1)
            p = torch.nan_to_num(torch.softmax(x, 1))[:, :L]
            off = 2.0 ** -9.7 / 7 * abs(scale) * (qh.abs().unflatten(1, (-1, 32)).sum(2) @ kh.abs().unflatten(1, (-1, 32)).amax(2).T)
            off = torch.where(seen, off, 0.0).amax(1, keepdim=True)
            tiles = torch.nn.functional.pad(vh.abs().amax(1), (0, -L % TILE)).view(-1, TILE).amax(1).repeat_interleave(TILE)[:L, None]
            groups = vh.abs().unflatten(1, (-1, 32)).amax(2).repeat_interleave(32, 1)
            if unpacked:
                floor = 2.0 ** -31 * (p * tiles[:, 0]).amax(1, keepdim=True) * (vh.abs() / torch.where(tiles > 0, tiles, 1.0)).sum(0)
            else:
                floor = 2.0 ** -30 * p.amax(1, keepdim=True) * tiles.max() * (vh.abs() / torch.where(groups > 0, groups, 1.0)).sum(0)
            ref, mass = p @ vh, p @ vh.abs()
            cols = slice(h * d, (h + 1) * d)
            out[t:t + n, cols] = ref
            bound[t:t + n, cols] = 2.0 ** -8 * ref.abs() + (2.0 ** -10 + 2 * off) * mass + floor
        t += n
    return out, bound
