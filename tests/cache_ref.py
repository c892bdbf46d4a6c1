"""The cache operators in 64 bits on the CPU, straight from their definitions (include/hoard_cache.h)."""
import math

import torch


def visibility(vis, m):
    """[m][m] bool: token t sees token i's row."""
    if vis is None:
        return torch.tril(torch.ones(m, m, dtype=torch.bool))
    return torch.tensor([[(int(w) >> i) & 1 for i in range(m)] for w in vis.tolist()], dtype=torch.bool).reshape(m, m)


def attention(q, k, v, n_past, vis=None, gate=None, scale=None, past_seen=None):
    """out [m][n_head][hd] and the weights' sums per KV head and row [n_kv][n], in 64 bits. past_seen [m][n_kv][n_past]:
    the past rows that are attended (default all). Rows that a token does not see take no part, whatever they hold."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    m, n_head, hd = q.shape
    n_kv = k.shape[1]
    n = n_past + m
    own = visibility(vis, m)
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(m, n_head, hd, dtype=torch.float64)
    acc = torch.zeros(n_kv, n, dtype=torch.float64)
    for h in range(n_head):
        kv = h * n_kv // n_head
        for t in range(m):
            past = torch.ones(n_past, dtype=torch.bool) if past_seen is None else past_seen[t, kv]
            rows = torch.cat([past, own[t]]).nonzero()[:, 0]
            if not len(rows):
                continue
            p = torch.softmax(k[rows, kv] @ q[t, h] * scale, 0)
            out[t, h] = p @ v[rows, kv]
            acc[kv, rows] += p
    if gate is not None:
        out *= torch.sigmoid(gate.double().cpu())
    return out, acc


def evict(k, v, acc, pos, n_rows, n_keep, n_sink, recent_from):
    """New (k, v, acc, pos), on the CPU, of one eviction in place."""
    k, v, acc, pos = (x.clone().cpu() for x in (k, v, acc, pos))
    for h in range(acc.shape[0]):
        def rank(j):
            if pos[h, j] < n_sink or pos[h, j] >= recent_from:
                return (0, 0.0, j)
            a = float(acc[h, j])
            return (2, 0.0, j) if math.isnan(a) else (1, -a, j)
        kept = set(sorted(range(n_rows), key=rank)[:n_keep])
        to = [j for j in range(n_keep) if j not in kept]
        frm = [j for j in range(n_keep, n_rows) if j in kept]
        for a, b in zip(to, frm):
            k[a, h], v[a, h], acc[h, a], pos[h, a] = k[b, h].clone(), v[b, h].clone(), acc[h, b].clone(), pos[h, b].clone()
    return k, v, acc, pos


def blocks(q, k, n_past, block, n_sink, n_local, n_sel):
    """chosen [m][n_kv] lists of block ids, and past_seen [m][n_kv][n_past]."""
    q, k = q.double().cpu(), k.double().cpu()
    m, n_head, _ = q.shape
    n_kv = k.shape[1]
    g = n_head // n_kv
    nb = -(-n_past // block)
    first, last = min(n_sink, nb), max(min(n_sink, nb), nb - n_local)
    at = torch.arange(n_past) // block
    seen = torch.zeros(m, n_kv, n_past, dtype=torch.bool)
    chosen = []
    for t in range(m):
        chosen.append([])
        for kv in range(n_kv):
            sel = []
            if last > first:
                kb = k[first * block:last * block, kv].reshape(last - first, block, -1)
                lo, hi = kb.amin(1), kb.amax(1)
                best = torch.full((last - first,), -math.inf, dtype=torch.float64)
                for h in range(kv * g, kv * g + g):
                    u = torch.maximum(q[t, h] * lo, q[t, h] * hi).sum(1)
                    best = torch.maximum(best, u - u.max())
                order = torch.argsort(best, descending=True, stable=True)[:n_sel]
                sel = sorted((order + first).tolist())
            chosen[-1].append(sel)
            seen[t, kv] = (at < first) | (at >= last) | torch.isin(at, torch.tensor(sel, dtype=torch.long))
    return chosen, seen
