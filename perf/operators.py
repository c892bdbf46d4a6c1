"""Cases of the operators on a KV cache: attention of a tree of drafted tokens, attention that accumulates its
weights, eviction by those weights, and attention over blocks of the cache that a score selects.

The caches are [row][KV head][head_dim] of f16 or bf16 values, activations are f32, as in the decode harness. Head
layouts are those of the benchmark configurations (32 / 4 heads of 128, 16 / 16 of 128, 16 / 2 of 256 with an output
gate) and generic ones.
"""
import math

import torch

own = False

KV = {"f16": torch.float16, "bf16": torch.bfloat16}
LAYOUTS = [(32, 4, 128, False), (16, 16, 128, False), (16, 2, 256, True), (8, 8, 64, False), (24, 4, 96, False),
           (12, 2, 80, False), (28, 4, 128, True), (6, 3, 256, False)]
MOST_ROWS = 1 << 27         # largest n * n_kv * head_dim of any case
MOST_FLOPS = 4 * 64 * 32 * 131072 * 128


def _attend(name, op, layout, n_past, m, kv, tree, **more):
    n_head, n_kv, hd, gate = layout
    return ({"name": name} if name else {}) | {"op": op, "n_head": n_head, "n_kv": n_kv, "head_dim": hd, "gate": gate,
                                               "n_past": n_past, "m": m, "kv": kv, "tree": tree} | more


def _evict(name, n_kv, hd, kv, n_rows, n_keep, n_sink, n_recent):
    return ({"name": name} if name else {}) | {"op": "evict", "n_kv": n_kv, "head_dim": hd, "kv": kv, "n_rows": n_rows,
                                               "n_keep": n_keep, "n_sink": n_sink, "n_recent": n_recent}


def listed():
    qwen3, olmoe, next80 = (32, 4, 128, False), (16, 16, 128, False), (16, 2, 256, True)
    return [
        # the first verify pass after a short prompt: latency
        _attend("tree short", "tree", qwen3, 37, 5, "f16", True),
        # a chain of drafts (the speculative loop's batch of 16) in an ordinary conversation
        _attend("chain of 16", "tree", qwen3, 4095, 16, "bf16", False),
        # multi-head layout: one query head per KV head, a wide tree
        _attend("tree, 16 KV heads", "tree", olmoe, 2011, 33, "f16", True),
        # a full tree of 64 drafts over a long document: matrix products
        _attend("tree of 64, long", "tree", qwen3, 131008, 64, "f16", True),
        # one token of a gated layer over a long cache
        _attend("token, gated, long", "tree", next80, 32769, 1, "bf16", False),
        # decode over a bounded cache: weights accumulated at each step
        _attend("weigh, bounded", "weigh", qwen3, 2303, 1, "bf16", False),
        # the same at the end of a long prompt, before its first eviction
        _attend("weigh, prompt", "weigh", olmoe, 30000, 1, "f16", False),
        # the eviction of a decode loop: every 256 tokens
        _evict("evict 2304 to 2048", 4, 128, "bf16", 2304, 2048, 4, 128),
        # a long prompt's cache brought down to its budget
        _evict("evict 65521 to 4096", 16, 128, "f16", 65521, 4096, 4, 1024),
        # the first token after a prompt: the blocks' bounds are formed, then used
        _attend("blocks, first token", "sparse", qwen3, 32767, 1, "bf16", False, block=64, n_sink=1, n_local=4, n_sel=32, build=True),
        # decode in a very long cache
        _attend("blocks, very long", "sparse", next80, 262081, 1, "f16", False, block=64, n_sink=1, n_local=8, n_sel=64, build=False),
        # a small tree verified over selected blocks
        _attend("blocks, tree of 8", "sparse", qwen3, 50001, 8, "f16", True, block=32, n_sink=2, n_local=4, n_sel=24, build=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weigh", "evict", "sparse"])
    layout = rng.choice(LAYOUTS)
    n_head, n_kv, hd, gate = layout
    kv = rng.choice(["f16", "bf16"])
    most = MOST_ROWS // (n_kv * hd)
    if op == "evict":
        n_rows = _log(rng, 2, min(100000, most))
        n_keep = rng.randint(max(1, n_rows // 16), n_rows - 1)
        n_sink = rng.randint(0, min(8, n_keep // 4))
        return _evict("", n_kv, hd, kv, n_rows, n_keep, n_sink, rng.randint(0, (n_keep - n_sink) // 2))
    if op == "weigh":
        return _attend("", op, layout, _log(rng, 1, min(100000, most)), 1, kv, False)
    if op == "tree":
        m = _log(rng, 1, 64)
        n_past = _log(rng, 1, min(131008, most - m, MOST_FLOPS // (4 * m * n_head * hd) - m))
        return _attend("", op, layout, n_past, m, kv, rng.random() < 0.7)
    m = _log(rng, 1, 16)
    block = rng.choice([16, 32, 64, 128])
    n_past = _log(rng, 100, min(262081, most - m))
    return _attend("", op, layout, n_past, m, kv, rng.random() < 0.7, block=block, n_sink=rng.randint(0, 2),
                   n_local=rng.randint(1, 8), n_sel=_log(rng, 4, 2048 // block), build=rng.random() < 0.3)


def _tree(case, seed):
    """Bit i of entry t: drafted token t sees drafted token i (itself and its ancestors; a token's parent is an earlier
    one, or the last token of the past)."""
    m = case["m"]
    g = torch.Generator().manual_seed(seed)
    vis = []
    for t in range(m):
        back = int(torch.randint(1, 5, (1,), generator=g))
        vis.append((vis[t - back] if case["tree"] and t - back >= 0 else vis[t - 1] if t and not case["tree"] else 0) | 1 << t)
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in vis], dtype=torch.int64).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_kv, hd, kt = case["n_kv"], case["head_dim"], KV[case["kv"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "evict":
        n, keep = case["n_rows"], case["n_keep"]
        s = {"case": case, "k": normal(n, n_kv, hd).to(kt), "v": normal(n, n_kv, hd).to(kt)}
        # weights: heavy-tailed, some rows never looked at (ties)
        acc = torch.exp(2.5 * normal(n_kv, n))
        s["acc"] = torch.where(torch.rand(n_kv, n, generator=g, device="cuda") < 0.2, torch.zeros_like(acc), acc)
        # positions: rows below n_keep in any order (earlier evictions), the others appended since
        pos = torch.arange(n, device="cuda", dtype=torch.int32).repeat(n_kv, 1)
        mix = torch.rand(n_kv, keep, generator=g, device="cuda").argsort(1)
        pos[:, :keep] = pos[:, :keep].gather(1, mix)
        s["pos"] = pos.contiguous()
        s["acc_out"], s["pos_out"] = torch.zeros_like(s["acc"]), torch.zeros_like(s["pos"])
        if own:
            from hoard_b200 import cache
            s["cache"] = cache.CacheOps(n_head=n_kv, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=n)
        return s
    m, n = case["m"], case["n_past"] + case["m"]
    rows = -(-n // 128) * 128           # the cache's rows: past the last token they hold what an earlier sequence left
    # keys with a part that drifts over the sequence, so that blocks differ, and channels of different size
    size = torch.exp(0.5 * normal(n_kv, hd))
    drift = normal(-(-rows // 96), n_kv, hd).repeat_interleave(96, 0)[:rows]
    k = ((normal(rows, n_kv, hd) + 0.7 * drift) * size).to(kt)
    s = {"case": case, "k": k, "v": normal(rows, n_kv, hd).to(kt)}
    s["q"] = 1.2 * normal(m, case["n_head"], hd) / size.repeat_interleave(case["n_head"] // n_kv, 0)
    s["gate"] = normal(m, case["n_head"], hd) if case["gate"] else None
    s["vis"] = _tree(case, seed)
    s["scale"] = 1.0 / math.sqrt(hd)
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "weigh":
        s["acc"] = torch.rand(n_kv, rows, generator=g, device="cuda")
    if case["op"] == "sparse":
        s["bounds"] = _bounds(k, case["block"])
        s["sel"] = torch.empty(m, n_kv, case["n_sel"], dtype=torch.int32, device="cuda")
    if own:
        from hoard_b200 import cache
        s["cache"] = cache.CacheOps(n_head=case["n_head"], n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=rows,
                                    max_tokens=m, block=case.get("block", 64))
    return s


def _bounds(k, block):
    """[KV head][block][min, max][head_dim] of the cache's complete blocks."""
    nb = k.shape[0] // block
    b = k[: nb * block].view(nb, block, k.shape[1], k.shape[2])
    return torch.stack([b.amin(1), b.amax(1)], 2).transpose(0, 1).contiguous()


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        c = s["cache"]
        if op == "evict":
            c.evict(s["k"], s["v"], s["acc"], s["pos"], case["n_rows"], case["n_keep"], n_sink=case["n_sink"],
                    recent_from=case["n_rows"] - case["n_recent"], acc_out=s["acc_out"], pos_out=s["pos_out"])
            return [s["k"], s["v"], s["acc_out"], s["pos_out"]]
        if op == "tree":
            return c.tree_attention(s["q"], s["k"], s["v"], case["n_past"], vis=s["vis"], gate=s["gate"], out=s["out"])
        if op == "weigh":
            return [c.tree_attention(s["q"], s["k"], s["v"], case["n_past"], vis=s["vis"], gate=s["gate"], acc=s["acc"], out=s["out"]),
                    s["acc"]]
        if case["build"]:
            c.block_bounds(s["k"], s["bounds"], 0, case["n_past"])
        out = c.block_attention(s["q"], s["k"], s["v"], s["bounds"], case["n_past"], n_sink=case["n_sink"], n_local=case["n_local"],
                                n_sel=case["n_sel"], vis=s["vis"], gate=s["gate"], out=s["out"], sel_out=s["sel"])
        return [out, s["sel"], s["bounds"]]
    if op == "evict":
        return _plain_evict(s)
    if op == "sparse":
        return _plain_sparse(s)
    out, acc = _plain_dense(s)
    if op == "tree":
        return out
    s["acc"][:, : acc.shape[1]] += acc
    return [out, s["acc"]]


# ---- plain forms --------------------------------------------------------------------------------------------------

def _own_rows(s):
    """[m][m]: whether token t sees token i."""
    m = s["case"]["m"]
    return (s["vis"][:, None] >> torch.arange(m, device="cuda")) & 1 != 0


def _softmax(x):
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _gated(s, out):
    return out if s["gate"] is None else out / (1 + torch.exp(-s["gate"]))


def _plain_dense(s):
    c = s["case"]
    m, n_kv, hd, n = c["m"], c["n_kv"], c["head_dim"], c["n_past"] + c["m"]
    g = c["n_head"] // n_kv
    q = s["q"].view(m, n_kv, g, hd).permute(1, 0, 2, 3).reshape(n_kv, m * g, hd)
    k, v = (s[x][:n].float().transpose(0, 1) for x in "kv")
    x = (q @ k.transpose(1, 2) * s["scale"]).view(n_kv, m, g, n)
    x[..., c["n_past"]:].masked_fill_(~_own_rows(s)[:, None], -math.inf)
    p = _softmax(x)
    out = (p.view(n_kv, m * g, n) @ v).view(n_kv, m, g, hd).permute(1, 0, 2, 3).reshape(m, c["n_head"], hd)
    return _gated(s, out), p.sum((1, 2))


def _plain_evict(s):
    c = s["case"]
    n, keep, acc, pos = c["n_rows"], c["n_keep"], s["acc"], s["pos"]
    safe = (pos < c["n_sink"]) | (pos >= n - c["n_recent"])
    order = torch.where(safe, torch.full_like(acc, math.inf), acc).argsort(dim=1, descending=True, stable=True)
    kept = torch.zeros_like(safe).scatter_(1, order[:, :keep], True)
    most = min(keep, n - keep)
    to = kept[:, :keep].to(torch.uint8).argsort(dim=1, stable=True)[:, :most]
    frm = (~kept[:, keep:]).to(torch.uint8).argsort(dim=1, stable=True)[:, :most] + keep
    moves = torch.arange(most, device="cuda") < (~kept[:, :keep]).sum(1, keepdim=True)
    frm = torch.where(moves, frm, to)
    head = torch.arange(c["n_kv"], device="cuda")[:, None]
    for x in ("k", "v"):
        s[x][to, head] = s[x][frm, head]
    for x in ("acc", "pos"):
        s[x + "_out"][:, :keep] = s[x][:, :keep]
        s[x + "_out"].scatter_(1, to, s[x].gather(1, frm))
    return [s["k"], s["v"], s["acc_out"], s["pos_out"]]


def _plain_sparse(s):
    c = s["case"]
    m, n_kv, hd, past, block = c["m"], c["n_kv"], c["head_dim"], c["n_past"], c["block"]
    g = c["n_head"] // n_kv
    if c["build"]:
        s["bounds"][:, : past // block] = _bounds(s["k"][:past], block)
    nb = -(-past // block)
    first, last = min(c["n_sink"], nb), max(min(c["n_sink"], nb), nb - c["n_local"])
    q = s["q"].view(m, n_kv, g, hd).permute(1, 0, 2, 3)
    if last > first:        # candidates: the blocks' scores decide which rows are read, so they are formed in 64 bits
        q2 = q.reshape(n_kv, m * g, hd).double()
        low, high = s["bounds"][:, first:last].double().unbind(2)
        u = q2.clamp(min=0) @ high.transpose(1, 2) + q2.clamp(max=0) @ low.transpose(1, 2)
        score = (u - u.amax(2, keepdim=True)).view(n_kv, m, g, -1).amax(2)
        sel = score.argsort(dim=2, descending=True, stable=True)[..., : c["n_sel"]].sort(2).values + first
    else:
        sel = torch.empty(n_kv, m, 0, dtype=torch.int64, device="cuda")
    s["sel"].fill_(-1)
    s["sel"][..., : sel.shape[2]] = sel.transpose(0, 1).to(torch.int32)
    always = torch.cat([torch.arange(first, device="cuda"), torch.arange(last, nb, device="cuda")])
    blocks = torch.cat([sel, always.expand(n_kv, m, -1)], 2)
    rows = (blocks[..., None] * block + torch.arange(block, device="cuda")).view(n_kv, m, -1)
    there = rows < past
    rows = torch.cat([torch.where(there, rows, torch.zeros_like(rows)), torch.arange(past, past + m, device="cuda").expand(n_kv, m, m)], 2)
    there = torch.cat([there, _own_rows(s).expand(n_kv, m, m)], 2)
    head = torch.arange(n_kv, device="cuda")[:, None, None]
    k, v = (s[x][rows, head].float() for x in "kv")
    x = q @ k.transpose(2, 3) * s["scale"]
    p = _softmax(x.masked_fill(~there[:, :, None], -math.inf))
    out = (p @ v).permute(1, 0, 2, 3).reshape(m, c["n_head"], hd)
    return [_gated(s, out), s["sel"], s["bounds"]]


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        # values only move; weights and positions are looked up head by head
        k, v, acc_out, pos_out = s["k"].clone(), s["v"].clone(), s["acc_out"].double(), s["pos_out"].clone()
        keep, n = case["n_keep"], case["n_rows"]
        acc, pos = s["acc"].double().cpu(), s["pos"].cpu()
        for h in range(case["n_kv"]):
            value = [math.inf if p < case["n_sink"] or p >= n - case["n_recent"] else a for a, p in zip(acc[h].tolist(), pos[h].tolist())]
            chosen = set(sorted(range(n), key=lambda j: (-value[j], j))[:keep])
            to = torch.tensor([j for j in range(keep) if j not in chosen], dtype=torch.long, device="cuda")
            frm = torch.tensor([j for j in range(keep, n) if j in chosen], dtype=torch.long, device="cuda")
            where = torch.arange(keep, device="cuda")
            where[to] = frm
            k[:keep, h], v[:keep, h] = s["k"][where, h], s["v"][where, h]
            acc_out[h, :keep], pos_out[h, :keep] = s["acc"][h, where].double(), s["pos"][h, where]
        return [k.double(), v.double(), acc_out, pos_out]
    m, hd, past = case["m"], case["head_dim"], case["n_past"]
    g, n = case["n_head"] // case["n_kv"], past + m
    vis = s["vis"].tolist()
    own_part = torch.tensor([[vis[t] >> i & 1 for i in range(m)] for t in range(m)], dtype=torch.bool, device="cuda")
    out = torch.empty(m, case["n_head"], hd, dtype=torch.float64, device="cuda")
    seen = torch.cat([torch.ones(m, past, dtype=torch.bool, device="cuda"), own_part], 1)
    weights = s["acc"].double() if case["op"] == "weigh" else None
    for h in range(case["n_head"]):
        kv = h // g
        if case["op"] == "sparse" and h % g == 0:
            seen = torch.cat([_exact_blocks(case, s, kv), own_part], 1)
        z = s["q"][:, h].double() @ s["k"][:n, kv].double().T * s["scale"]
        p = torch.softmax(z.masked_fill(~seen, -math.inf), 1)
        out[:, h] = p @ torch.where(seen.any(0)[:, None], s["v"][:n, kv].double(), 0.0)
        if s["gate"] is not None:
            out[:, h] *= torch.sigmoid(s["gate"][:, h].double())
        if weights is not None:
            weights[kv, :n] += p.sum(0)
    if case["op"] == "tree":
        return out
    return [out, weights] if weights is not None else [out, None, None]


def _exact_blocks(case, s, kv):
    """[m][n_past]: the past rows that each token attends in KV head kv."""
    m, past, block, g = case["m"], case["n_past"], case["block"], case["n_head"] // case["n_kv"]
    at = torch.arange(past, device="cuda") // block
    nb = -(-past // block)
    always = (at < case["n_sink"]) | (at >= nb - case["n_local"])
    inner = list(range(case["n_sink"], nb - case["n_local"]))
    if not inner:
        return always.expand(m, past)
    k = s["k"][inner[0] * block: (inner[-1] + 1) * block, kv].double().view(len(inner), block, -1)
    seen = []
    for t in range(m):
        best = None
        for h in range(kv * g, kv * g + g):
            q = s["q"][t, h].double()
            u = torch.maximum(q * k.amin(1), q * k.amax(1)).sum(1)
            u = u - u.max()
            best = u if best is None else torch.maximum(best, u)
        best = best.tolist()
        chosen = sorted(range(len(inner)), key=lambda b: (-best[b], b))[: case["n_sel"]]
        seen.append(always | torch.isin(at, torch.tensor([inner[b] for b in chosen], device="cuda")))
    return torch.stack(seen)


def work(case):
    n_kv, hd = case["n_kv"], case["head_dim"]
    if case["op"] == "evict":
        # the weights and positions once, the kept ones out; about as many rows move as would by an even choice
        n, keep = case["n_rows"], case["n_keep"]
        moved = (n - keep) * keep / n
        return {"bytes": 8 * n_kv * (n + keep) + moved * n_kv * hd * 2 * 2 * 2, "flops": 0}
    m, past = case["m"], case["n_past"]
    rows, more = past + m, 0
    if case["op"] == "sparse":
        block = case["block"]
        nb = -(-past // block)
        rows = min(rows, (case["n_sink"] + case["n_local"] + case["n_sel"]) * block + m)
        more = 4 * n_kv * hd * nb + (2 * n_kv * hd * past if case["build"] else 0)
    acts = 4 * m * case["n_head"] * hd * (3 if case["gate"] else 2) + (8 * n_kv * rows if case["op"] == "weigh" else 0)
    return {"bytes": 4 * rows * n_kv * hd + acts + more, "flops": 4 * m * case["n_head"] * rows * hd}
