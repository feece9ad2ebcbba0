"""Plain forms of beam search's operators, on the CPU: lists and 64-bit numbers, one request and one row at a time."""
import math

import numpy as np
import torch


def select(logits, scores, k):
    """[(parents, tokens, scores)] of every request, and the flags of its rows."""
    R, W = scores.shape
    V = logits.shape[1]
    x = logits.double().cpu().numpy()
    base_scores = scores.double().cpu().numpy()
    found, bad = [], []
    for r in range(R):
        flats, ss, xs = [], [], []
        for w in range(W):
            row = x[r * W + w]
            broken = bool(np.isnan(row).any() or (row == np.inf).any())
            bad.append(int(broken))
            if broken or not np.isfinite(base_scores[r, w]) or np.isinf(row).all():
                continue
            m = row.max()
            base = base_scores[r, w] - (m + math.log(np.exp(row - m).sum()))
            at = np.nonzero(row > -np.inf)[0]
            flats.append(w * V + at)
            ss.append(base + row[at])
            xs.append(row[at])
        if flats:
            flat, s, xx = (np.concatenate(a) for a in (flats, ss, xs))
            order = np.lexsort((flat, -xx, -s))[:k]
            flat, s = flat[order], s[order]
        else:
            flat, s = np.zeros(0, np.int64), np.zeros(0)
        pad = k - len(flat)
        found.append((np.concatenate([flat // V, np.full(pad, -1)]).tolist(), np.concatenate([flat % V, np.full(pad, -1)]).tolist(),
                      np.concatenate([s, np.full(pad, -np.inf)]).tolist()))
    return found, bad


def places(parents):
    """Whose place each child takes, and whose rows are copied there (None: nobody's)."""
    W = len(parents)
    got, source, taken = [None] * W, [None] * W, set()
    for w, p in enumerate(parents):
        if p >= 0 and p not in taken:
            taken.add(p)
            got[w] = p
    free = [b for b in range(W) if b not in taken]
    for w, p in enumerate(parents):
        if got[w] is None:
            got[w] = free.pop(0)
            source[w] = p if p >= 0 else None
    return got, source


def reorder(parents, kv_len, groups, slots, states):
    """groups: [(table, [storages with pages on axis -4], page size, stride, rows of a unit)], all changed in place (tensors on the CPU)."""
    R, W = parents.shape
    new_slots = slots.clone() if slots is not None else None
    for r in range(R):
        par = parents[r].tolist()
        got, source = places(par)
        n = int(kv_len[r * W])
        for table, storages, page, stride, unit in groups:
            have = n // stride
            fill, last = have % page, have // page
            old = table[r * W:(r + 1) * W].clone()
            for w in range(W):
                if source[w] is not None and fill and last < table.shape[1]:
                    a, b = int(old[source[w], last]), int(old[got[w], last])
                    for x in storages:
                        if 0 <= a < x.shape[-4] and 0 <= b < x.shape[-4]:
                            x[..., b, :, :-(-fill // unit), :] = x[..., a, :, :-(-fill // unit), :]
                for c in range(min(table.shape[1], last + (fill > 0))):
                    table[r * W + w, c] = old[got[w], c] if (c == last and fill) else old[par[w] if par[w] >= 0 else w, c]
        if slots is not None:
            for w in range(W):
                new_slots[r * W + w] = slots[r * W + got[w]]
                if source[w] is not None:
                    a, b = int(slots[r * W + source[w]]), int(slots[r * W + got[w]])
                    for x in states:
                        x[b] = x[a]
    if slots is not None:
        slots.copy_(new_slots)


def build(new, cached, groups):
    """(cu_q, kv_len, positions, seq, slot map); groups: [[table, free, used, page, stride]] (lists), whose tables and used change."""
    cu, positions, seq = [0], [], []
    for s, (n, c) in enumerate(zip(new, cached)):
        cu.append(cu[-1] + n)
        positions += list(range(c, c + n))
        seq += [s] * n
    for g in groups:
        table, free, used, page, stride = g
        for s, (n, c) in enumerate(zip(new, cached)):
            for b in range(-(-(c // stride) // page), -(-((c + n) // stride) // page)):
                table[s][b] = free[used]
                used += 1
        g[2] = used
    slot_map = []
    if groups:
        table, _, _, page, _ = groups[0]
        for s, p in zip(seq, positions):
            at = table[s][p // page]
            slot_map.append(at * page + p % page if at >= 0 else -1)
    return cu, [n + c for n, c in zip(new, cached)], positions, seq, slot_map


def keep(cands, stops, W, step, last, penalty, early, state):
    """One request.  cands: [(parent, token, score)] best first; state: dict(done [(score, step, parent, token)], over).  Returns the beams that go on."""
    live = []
    length = float(step + 1) ** penalty
    over = state["over"]

    def add(score, parent, token):
        done = state["done"]
        if len(done) == W and not score > done[-1][0]:
            return
        done.append((score, step, parent, token))
        done.sort(key=lambda d: -d[0])            # (stable: an earlier one stays before an equal later one)
        del done[W:]

    ends = []
    for i, (parent, token, score) in enumerate(cands):
        if parent < 0:
            break
        if token in stops:
            if i < W:
                ends.append((i, score, parent, token))
        elif len(live) < W:
            live.append((parent, token, score))
            if step + 1 >= last:
                ends.append((i, score, parent, token))
    if not over:
        for _, score, parent, token in sorted(ends):
            add(score / length, parent, token)
        best = cands[0][2] if cands and cands[0][0] >= 0 else -math.inf
        if not live or step + 1 >= last or (len(state["done"]) == W and (early or not best / length > state["done"][-1][0])):
            state["over"] = True
    return live


def attention(q, k_cache, v_cache, positions, table, window, scale, nq, nkv, sink=None):
    """[rows, nq * d] in 64 bits, and for each (row, head) the largest |score| and the sum of p |v| at each element (what a bound needs)."""
    rows, d, page = q.shape[0], q.shape[1] // nq, k_cache.shape[2]
    out, mass = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    most = torch.zeros(rows, nq, dtype=torch.float64)
    q, k_cache, v_cache, table = q.double().cpu(), k_cache.double().cpu(), v_cache.double().cpu(), table.cpu()
    for i in range(rows):
        pos = int(positions[i])
        if pos < 0:
            continue
        lo = max(0, pos + 1 - window) if window > 0 else pos - pos % -window if window < 0 else 0
        at = torch.arange(lo, max(lo, min(pos + 1, table.shape[1] * page)))
        ids = table[i, at // page].long()
        at, ids = at[(ids >= 0) & (ids < k_cache.shape[0])], ids[(ids >= 0) & (ids < k_cache.shape[0])]
        k, v = k_cache[ids, :, at % page], v_cache[ids, :, at % page]
        for h in range(nq):
            x = k[:, h // (nq // nkv)] @ q[i, h * d:(h + 1) * d] * scale
            if sink is not None:
                x = torch.cat([x, sink[h:h + 1].double().cpu()])
            if x.numel() == 0:
                continue
            p = torch.softmax(x, 0)[:at.numel()]
            if at.numel():
                out[i, h * d:(h + 1) * d] = p @ v[:, h // (nq // nkv)]
                mass[i, h * d:(h + 1) * d] = p @ v[:, h // (nq // nkv)].abs()
                most[i, h] = (k[:, h // (nq // nkv)].abs() @ q[i, h * d:(h + 1) * d].abs() * abs(scale)).max()
    return out, mass, most
