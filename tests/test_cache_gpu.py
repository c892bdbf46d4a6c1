"""The cache operators (hoard_b200/cache.py) against their definitions in 64 bits (tests/cache_ref.py).

Tolerances. Outputs are f32 sums of weights p (relative error e_p) times stored values. With u = 2^-24 (half a step
of f32): a score of magnitude s (in units of log2) is a sum of at most 16 K-step sums, each of products that are exact to
2^-22 (two f16 terms) or better, rounded or truncated once per K step: |error| <= (16 + 4) u |s|_max, and the weight's
relative error is ln 2 times that, plus 2^-22 for the exponential. Scores here stay below |s| = 32, so e_p <= 20 * 32 *
0.7 u + 4 u < 460 u = 2.8e-5 in the worst case; errors of different rows are independent, and the norm-wise error that is
tested is their root mean square, an eighth of that at most: 4e-6 over all outputs. Accumulated weights: the same."""
import ctypes

import pytest
import torch

from hoard_b200 import cache
from hoard_b200.moe import HoardError
from tests import cache_ref as ref

pytestmark = pytest.mark.gpu
TOL = 4e-6
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / max(float(b.norm()), 1e-300))


def case(n_head, n_kv, hd, kt, rows, m, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    size = torch.exp(0.4 * r(n_kv, hd))
    k, v = (r(rows, n_kv, hd) * size).to(kt), r(rows, n_kv, hd).to(kt)
    q = r(m, n_head, hd) / size.repeat_interleave(n_head // n_kv, 0)
    return q, k, v, r


def tree(m, seed):
    g = torch.Generator().manual_seed(seed)
    parents = [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(m)]
    words, depth = cache.tree_visibility(parents)
    return torch.tensor(words, dtype=torch.int64, device=DEV), parents


LAYOUTS = [(8, 2, 128), (4, 4, 64), (16, 1, 256), (6, 2, 80), (3, 3, 8), (12, 2, 96), (64, 1, 40)]


@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("n_head,n_kv,hd", LAYOUTS)
@pytest.mark.parametrize("n_past,m", [(0, 1), (0, 7), (1, 1), (15, 2), (16, 16), (47, 5), (300, 33), (1000, 64), (2049, 1)])
def test_tree_attention(n_head, n_kv, hd, kt, n_past, m):
    q, k, v, r = case(n_head, n_kv, hd, kt, n_past + m + 3, m, seed=n_past + m)
    vis, _ = tree(m, n_past)
    k[n_past + m:], v[n_past + m:] = float("nan"), float("nan")          # rows behind the last token are not read
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=n_past + m + 3, max_tokens=m)
    out = ops.tree_attention(q, k, v, n_past, vis=vis)
    want, _ = ref.attention(q, k, v, n_past, vis)
    assert rel(out, want) < TOL
    chain = ops.tree_attention(q, k, v, n_past)
    assert rel(chain, ref.attention(q, k, v, n_past)[0]) < TOL


@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("n_head,n_kv,hd,m", [(32, 4, 128, 16), (16, 16, 128, 40), (8, 8, 64, 64), (24, 4, 96, 11), (12, 2, 80, 64)])
@pytest.mark.parametrize("n_past", [513, 4000])
def test_tree_attention_many_rows(n_head, n_kv, hd, m, kt, n_past):
    """More query rows per KV head than the tensor-core form's threshold."""
    q, k, v, _ = case(n_head, n_kv, hd, kt, n_past + m, m, seed=m)
    vis, _ = tree(m, m)
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=n_past + m, max_tokens=m)
    out = ops.tree_attention(q, k, v, n_past, vis=vis)
    kd, vd, qd = k.double(), v.double(), q.double()
    g = n_head // n_kv
    own = ref.visibility(vis, m).to(DEV)
    x = torch.einsum("tkgd,jkd->tkgj", qd.view(m, n_kv, g, hd), kd) / hd**0.5
    x[..., n_past:].masked_fill_(~own[:, None, None, :], float("-inf"))
    want = torch.einsum("tkgj,jkd->tkgd", torch.softmax(x, -1), vd).reshape(m, n_head, hd)
    assert rel(out, want) < TOL


@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("n_past,m", [(0, 4), (40, 20), (700, 20)])
def test_masked_rows_may_hold_anything(kt, n_past, m):
    """Infinities and NaN in K and V of rows that a token does not see leave its output alone; who sees them gets them."""
    q, k, v, _ = case(8, 2, 128, kt, n_past + m, m)
    vis, _ = tree(m, 3)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=kt, max_rows=n_past + m, max_tokens=m)
    clean = ops.tree_attention(q, k, v, n_past, vis=vis)
    bad = m - 2
    sees = ref.visibility(vis, m)[:, bad].to(DEV)
    for value in (float("inf"), float("-inf"), float("nan")):
        k2, v2 = k.clone(), v.clone()
        v2[n_past + bad, :, ::2] = value
        out = ops.tree_attention(q, k, v2, n_past, vis=vis)
        assert rel(out[~sees], clean[~sees]) < TOL and not torch.isfinite(out[sees][..., ::2]).any()
        k2[n_past + bad] = value
        out = ops.tree_attention(q, k2, v2, n_past, vis=vis)
        assert rel(out[~sees], clean[~sees]) < TOL
    # lowest finite values are values, not masks
    low = torch.finfo(kt).min
    k2 = k.clone()
    k2[n_past + bad] = low if kt is BF16 else -1000.0
    out = ops.tree_attention(q, k2, v, n_past, vis=vis)
    assert rel(out[~sees], clean[~sees]) < TOL


@pytest.mark.parametrize("kt", [F16, BF16])
def test_token_that_sees_nothing(kt):
    q, k, v, _ = case(8, 2, 128, kt, 8, 8)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=kt, max_rows=8, max_tokens=8)
    vis = torch.tensor([0, 1, 2, 0, 5, 0, 64, 128], dtype=torch.int64, device=DEV)
    out = ops.tree_attention(q, k, v, 0, vis=vis)
    want, _ = ref.attention(q, k, v, 0, vis)
    assert rel(out, want) < TOL and out[0].abs().max() == 0 and out[3].abs().max() == 0


@pytest.mark.parametrize("n_past,m", [(30, 5), (900, 20), (900, 64)])
def test_visibility_bits_beyond_the_tokens(n_past, m):
    q, k, v, _ = case(8, 2, 128, F16, n_past + m + 64, m)
    k[n_past + m:], v[n_past + m:] = float("nan"), float("nan")
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=n_past + m + 64, max_tokens=m)
    every = torch.full((m,), -1, dtype=torch.int64, device=DEV)
    just = torch.full((m,), (1 << m) - 1 if m < 64 else -1, dtype=torch.int64, device=DEV)
    out = ops.tree_attention(q, k, v, n_past, vis=every)
    assert torch.equal(out, ops.tree_attention(q, k, v, n_past, vis=just)) and torch.isfinite(out).all()


@pytest.mark.parametrize("n_past,m", [(30, 3), (900, 20)])
def test_nan_query_stays_in_its_row(n_past, m):
    q, k, v, _ = case(8, 2, 128, F16, n_past + m, m)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=n_past + m, max_tokens=m)
    clean = ops.tree_attention(q, k, v, n_past)
    q2 = q.clone()
    q2[1, 5] = float("nan")
    out = ops.tree_attention(q2, k, v, n_past)
    assert torch.isnan(out[1, 5]).all()
    out[1, 5] = clean[1, 5]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("scale_q,scale_k", [(1e-20, 1.0), (1e4, 1e-4), (1e-30, 1.0)])
def test_extreme_magnitudes(scale_q, scale_k):
    q, k, v, _ = case(8, 2, 64, F16, 200, 2)
    q, k = q * scale_q, (k.float() * scale_k).half()
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=64, kv_dtype=F16, max_rows=200, max_tokens=2)
    assert rel(ops.tree_attention(q, k, v, 198), ref.attention(q, k, v, 198)[0]) < TOL


@pytest.mark.parametrize("m,n_past", [(2, 198), (20, 900)])
def test_queries_near_the_largest_float(m, n_past):
    """1.5 * 2^127 beside 2^120, over keys that bring the scores back to ordinary size."""
    q, k, v, r = case(8, 2, 64, BF16, n_past + m, m)
    q, k = q * 2.0**120, (k.float() * 2.0**-120).to(BF16)
    q[:, :, 0] = 1.5 * 2.0**127 * torch.sign(q[:, :, 0])
    k[:, :, 0] = (r(n_past + m, 2) * 2.0**-124).to(BF16)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=64, kv_dtype=BF16, max_rows=n_past + m, max_tokens=m)
    assert rel(ops.tree_attention(q, k, v, n_past), ref.attention(q, k, v, n_past)[0]) < TOL


@pytest.mark.parametrize("m,n_past", [(3, 40), (3, 3000), (20, 900)])
def test_head_major_queries_and_output_in_place(m, n_past):
    """q as [n_head][m][head_dim]'s transpose; out the same tensor as q: results to the bit."""
    q, k, v, r = case(8, 2, 128, F16, n_past + m, m)
    gate = r(8, m, 128).transpose(0, 1)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=n_past + m, max_tokens=m, block=16)
    bounds = torch.zeros(2, (n_past + m) // 16, 2, 128, dtype=F16, device=DEV)
    ops.block_bounds(k, bounds, 0, n_past)
    major = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert major.stride()[1] == m * 128
    for call in (lambda q, **kw: ops.tree_attention(q, k, v, n_past, gate=gate, **kw),
                 lambda q, **kw: ops.block_attention(q, k, v, bounds, n_past, n_sink=1, n_local=1, n_sel=2, **kw)):
        want = call(q)
        assert torch.equal(call(major), want)
        x = q.clone()
        assert call(x, out=x) is x and torch.equal(x, want)


@pytest.mark.parametrize("m,n_past", [(1, 77), (20, 900)])
def test_strides_gate_and_layouts(m, n_past):
    """q and gate inside wider rows, a cache laid out [head][row][dim], an output that is given."""
    n_head, n_kv, hd = 8, 2, 128
    q, k, v, r = case(n_head, n_kv, hd, BF16, n_past + m, m)
    fused = r(m, n_head, 2 * hd + 3)
    fused[..., :hd] = q
    qs, gate = fused[..., :hd], fused[..., hd:2 * hd]
    kh, vh = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=BF16, max_rows=n_past + m, max_tokens=m)
    out = torch.full((m, n_head, hd), float("nan"), device=DEV)
    ops.tree_attention(qs, kh, vh, n_past, gate=gate, out=out)
    want, _ = ref.attention(q, k, v, n_past, gate=gate)
    assert rel(out, want) < TOL
    # the same object with the other layout again
    assert rel(ops.tree_attention(qs, k, v, n_past, gate=gate), want) < TOL


@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("n_head,n_kv,hd,m,n_past", [(8, 2, 128, 1, 0), (8, 2, 128, 1, 40), (4, 4, 64, 1, 2500), (16, 2, 256, 1, 700),
                                                     (8, 2, 128, 5, 333), (64, 1, 40, 3, 100)])
def test_accumulated_weights(n_head, n_kv, hd, kt, m, n_past):
    q, k, v, r = case(n_head, n_kv, hd, kt, n_past + m + 5, m)
    vis, _ = tree(m, 1)
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=n_past + m + 5, max_tokens=m,
                         max_acc_tokens=m)
    acc0 = torch.rand(n_kv, n_past + m + 5, device=DEV)
    acc = acc0.clone()
    out = ops.tree_attention(q, k, v, n_past, vis=vis, acc=acc)
    want, add = ref.attention(q, k, v, n_past, vis)
    assert rel(out, want) < TOL
    assert rel(acc[:, :n_past + m], acc0[:, :n_past + m].double().cpu() + add) < TOL
    assert torch.equal(acc[:, n_past + m:], acc0[:, n_past + m:])
    # the same numbers every time
    acc2 = acc0.clone()
    assert torch.equal(ops.tree_attention(q, k, v, n_past, vis=vis, acc=acc2), out) and torch.equal(acc2, acc)


@pytest.mark.parametrize("n_rows,n_keep", [(1, 1), (2, 1), (33, 32), (100, 7), (1000, 999), (2304, 2048), (5000, 600),
                                           (10240, 10176), (10240, 10100), (10241, 10177), (40000, 37000), (70001, 3000)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict(n_rows, n_keep, kind):
    n_kv, hd, kt = 3, 64, F16
    g = torch.Generator(device=DEV).manual_seed(n_rows)
    rows = n_rows + 2
    k, v = (torch.randn(rows, n_kv, hd, generator=g, device=DEV).to(kt) for _ in range(2))
    acc = torch.exp(2 * torch.randn(n_kv, rows, generator=g, device=DEV))
    if kind == "ties":
        acc = torch.floor(acc).clamp(max=2)
    if kind == "odd":
        acc[:, ::5], acc[:, 1::7], acc[:, 2::9], acc[:, 3::11] = float("nan"), float("inf"), -0.0, -1.0
    pos = torch.stack([torch.randperm(rows, generator=g, device=DEV) for _ in range(n_kv)]).int()
    n_sink, recent_from = min(2, n_keep // 2), rows - n_keep // 3
    want = ref.evict(k, v, acc, pos, n_rows, n_keep, n_sink, recent_from)
    ops = cache.CacheOps(n_head=n_kv, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=rows)
    ao, po = acc.clone(), pos.clone()
    k1, v1 = k.clone(), v.clone()
    ops.evict(k1, v1, acc, pos, n_rows, n_keep, n_sink=n_sink, recent_from=recent_from, acc_out=ao, pos_out=po)
    ops.evict(k, v, acc, pos, n_rows, n_keep, n_sink=n_sink, recent_from=recent_from)           # in place
    for a, b, w in zip((k, v, acc, pos), (k1, v1, ao, po), want):
        assert torch.equal(a.cpu().view(torch.int16 if a.dtype is kt else torch.int32),
                           w.view(torch.int16 if a.dtype is kt else torch.int32))
        assert torch.equal(b.cpu().view(torch.int16 if a.dtype is kt else torch.int32),
                           w.view(torch.int16 if a.dtype is kt else torch.int32))


@pytest.mark.parametrize("n_rows,n_keep", [(140001, 70000), (330001, 5000)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_very_many_rows(n_rows, n_keep, ties):
    """More rows for each CTA of the cluster than one scan takes, and than its shared memory holds."""
    g = torch.Generator(device=DEV).manual_seed(n_rows)
    k, v = (torch.randn(n_rows, 2, 8, generator=g, device=DEV).half() for _ in range(2))
    acc = torch.exp(2 * torch.randn(2, n_rows, generator=g, device=DEV))
    if ties:
        acc = torch.floor(acc).clamp(max=2)
    pos = torch.arange(n_rows, device=DEV, dtype=torch.int32).repeat(2, 1)
    want = ref.evict(k, v, acc, pos, n_rows, n_keep, 4, n_rows - 100)
    ops = cache.CacheOps(n_head=2, n_head_kv=2, head_dim=8, kv_dtype=F16, max_rows=n_rows)
    ops.evict(k, v, acc, pos, n_rows, n_keep, n_sink=4, recent_from=n_rows - 100)
    for a, w in zip((k, v, acc, pos), want):
        assert torch.equal(a.cpu(), w)


def test_evict_more_protected_rows_than_are_kept():
    n_kv, hd, rows = 2, 16, 50
    k = torch.arange(rows, device=DEV).half()[:, None, None].expand(rows, n_kv, hd).contiguous()
    acc = torch.rand(n_kv, rows, device=DEV)
    pos = torch.arange(rows, device=DEV, dtype=torch.int32).repeat(n_kv, 1)
    ops = cache.CacheOps(n_head=2, n_head_kv=2, head_dim=hd, kv_dtype=F16, max_rows=rows)
    v = k.clone()
    ops.evict(k, v, acc, pos, rows, 10, n_sink=30)
    assert torch.equal(pos[:, :10].cpu(), torch.arange(10, dtype=torch.int32).repeat(2, 1))     # the lower rows


@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("n_head,n_kv,hd,block,n_past,m", [(8, 2, 128, 16, 500, 1), (4, 4, 64, 64, 1000, 3), (16, 2, 256, 32, 777, 2),
                                                          (6, 2, 80, 128, 2000, 5), (64, 1, 40, 16, 333, 1), (8, 2, 128, 16, 5, 4),
                                                          (8, 2, 128, 64, 0, 2)])
@pytest.mark.parametrize("n_sink,n_local,n_sel", [(1, 1, 3), (0, 2, 0), (2, 3, 1000)])
def test_block_attention(n_head, n_kv, hd, kt, block, n_past, m, n_sink, n_local, n_sel):
    rows = n_past + m + 70
    q, k, v, _ = case(n_head, n_kv, hd, kt, rows, m, seed=block)
    vis, _ = tree(m, 2)
    k[n_past + m:], v[n_past + m:] = float("nan"), float("nan")
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=rows, max_tokens=m, block=block)
    bounds = torch.zeros(n_kv, rows // block, 2, hd, dtype=kt, device=DEV)
    half = n_past // 2
    ops.block_bounds(k, bounds, 0, half)
    ops.block_bounds(k, bounds, half, n_past)
    nb = n_past // block
    kb = k[:nb * block].view(nb, block, n_kv, hd)
    if nb:
        assert torch.equal(bounds[:, :nb, 0].transpose(0, 1), kb.amin(1)) and torch.equal(bounds[:, :nb, 1].transpose(0, 1), kb.amax(1))
    assert bounds[:, nb:].abs().max() == 0 if nb < rows // block else True
    sel = torch.full((m, n_kv, n_sel), 99, dtype=torch.int32, device=DEV)
    out = ops.block_attention(q, k, v, bounds, n_past, n_sink=n_sink, n_local=n_local, n_sel=n_sel, vis=vis, sel_out=sel)
    chosen, seen = ref.blocks(q, k, n_past, block, n_sink, n_local, n_sel)
    for t in range(m):
        for h in range(n_kv):
            assert sel[t, h].tolist() == chosen[t][h] + [-1] * (n_sel - len(chosen[t][h]))
    assert rel(out, ref.attention(q, k, v, n_past, vis, past_seen=seen)[0]) < TOL


@pytest.mark.parametrize("same", [1, 3])
def test_block_ties_go_to_the_lower_block(same):
    """Blocks with equal keys score equally, however many there are."""
    n_past, block, n_kv, hd = 40 * 16, 16, 2, 64
    q, k, v, _ = case(4, n_kv, hd, F16, n_past + 1, 1)
    k[:n_past] = k[:same * block].repeat(-(-40 // same), 1, 1)[:n_past]
    ops = cache.CacheOps(n_head=4, n_head_kv=n_kv, head_dim=hd, kv_dtype=F16, max_rows=n_past + 1, block=block)
    bounds = ops.block_bounds(k, torch.zeros(n_kv, 40, 2, hd, dtype=F16, device=DEV), 0, n_past)
    sel = torch.zeros(1, n_kv, 5, dtype=torch.int32, device=DEV)
    ops.block_attention(q, k, v, bounds, n_past, n_sink=1, n_local=1, n_sel=5, sel_out=sel)
    assert sel[0].tolist() == ref.blocks(q, k, n_past, block, 1, 1, 5)[0][0]


def test_many_blocks_take_the_cluster_path():
    n_past, block, n_kv, hd = 16 * 9000, 16, 1, 16
    q, k, v, _ = case(2, n_kv, hd, BF16, n_past + 1, 1)
    ops = cache.CacheOps(n_head=2, n_head_kv=n_kv, head_dim=hd, kv_dtype=BF16, max_rows=n_past + 1, block=block)
    bounds = ops.block_bounds(k, torch.zeros(n_kv, 9000, 2, hd, dtype=BF16, device=DEV), 0, n_past)
    sel = torch.zeros(1, n_kv, 100, dtype=torch.int32, device=DEV)
    out = ops.block_attention(q, k, v, bounds, n_past, n_sink=1, n_local=1, n_sel=100, sel_out=sel)
    chosen, seen = ref.blocks(q, k, n_past, block, 1, 1, 100)
    assert sel[0].tolist() == chosen[0]
    assert rel(out, ref.attention(q, k, v, n_past, past_seen=seen)[0]) < TOL


def test_take():
    rows, n_kv, hd, base = 90, 2, 40, 20
    k = torch.arange(rows, device=DEV).half()[:, None, None].expand(rows, n_kv, hd).contiguous()
    v = -k
    ops = cache.CacheOps(n_head=2, n_head_kv=n_kv, head_dim=hd, kv_dtype=F16, max_rows=rows)
    path = [0, 2, 3, 7, 8, 9, 10, 11, 12, 13, 20, 30, 31, 32, 33, 34, 35, 63]
    ops.take(k, v, base, path)
    want = list(range(rows))
    want[base:base + len(path)] = [base + p for p in path]
    assert k[:, 1, 3].tolist() == want and v[:, 0, 0].tolist() == [-x for x in want]
    ops.take(k, v, base, [])
    ops.take(k, v, base, [0, 1, 2])
    assert k[:, 1, 3].tolist() == want


@pytest.mark.parametrize("mode,gated,rope_dim", [(0, False, 128), (1, False, 128), (2, False, 128), (2, True, 64)])
def test_store_matches_the_single_token_form(mode, gated, rope_dim):
    """Bit for bit hoard_hx_qknorm_rope_store_ex where rows are positions; rows elsewhere hold the same values."""
    from hoard_b200 import harness as hx
    n_head, n_kv, hd, m, rows = 4, 2, 128, 5, 40
    g = torch.Generator(device=DEV).manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    qs = 2 * hd if gated else hd
    q, k, v = r(m, n_head, qs), r(m, n_kv, hd), r(m, n_kv, hd)
    qn, kn = (r(n_head * hd), r(n_kv * hd)) if mode == 1 else (r(hd), r(hd))
    pos = torch.tensor([9, 9, 10, 10, 11], dtype=torch.int32, device=DEV)
    kc, vc = (torch.zeros(rows, n_kv, hd, dtype=BF16, device=DEV) for _ in range(2))
    acc, row_pos = torch.ones(n_kv, rows, device=DEV), torch.full((n_kv, rows), -5, dtype=torch.int32, device=DEV)
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=BF16, max_rows=rows, max_tokens=m)
    rot = ops.store(q[:, :, :hd], k, v, kc, vc, pos, 30, q_norm=qn, k_norm=kn, mode=mode, rope_dim=rope_dim, freq_base=1e6,
                    acc=acc, row_pos=row_pos)
    k1, v1 = torch.zeros_like(kc), torch.zeros_like(vc)
    for t in range(m):
        one = torch.zeros(n_head, hd, device=DEV)
        hx._ok(hx._hx().hoard_hx_qknorm_rope_store_ex(q[t].data_ptr(), k[t].data_ptr(), v[t].data_ptr(), qn.data_ptr(),
                                                      kn.data_ptr(), mode, 1e-6, n_head, n_kv, hd, qs, rope_dim, int(pos[t]), None,
                                                      rows, 1e6, one.data_ptr(), k1.data_ptr(), v1.data_ptr(), 30, None), "store")
        assert torch.equal(rot[t], one)
        assert torch.equal(kc[30 + t], k1[int(pos[t])]) and torch.equal(vc[30 + t], v1[int(pos[t])])
    assert kc[:30].abs().max() == 0 and kc[35:].abs().max() == 0
    assert acc[:, 30:35].abs().max() == 0 and acc[:, :30].min() == 1 and acc[:, 35:].min() == 1
    assert row_pos[:, 30:35].tolist() == [pos.tolist()] * n_kv and (row_pos[:, :30] == -5).all()
    # rows outside the cache are not written
    before = kc.clone()
    dev_row = torch.tensor([rows - 1], dtype=torch.int32, device=DEV)
    ops.store(q[:, :, :hd], k, v, kc, vc, pos, row0_dev=dev_row, q_norm=qn, k_norm=kn, mode=mode, rope_dim=rope_dim, freq_base=1e6)
    assert torch.equal(kc[:rows - 1], before[:rows - 1]) and torch.equal(kc[rows - 1], before[30])


def test_device_position_in_a_replayed_graph():
    """One captured graph of store, attention with weights, block bounds and block attention, replayed at growing positions;
    two graphs with workspaces of their own, replayed in turn."""
    n_head, n_kv, hd, rows, block, steps = 8, 2, 128, 256, 16, 70
    q, k, v, r = case(n_head, n_kv, hd, F16, rows, 1)
    kin, vin, qin = r(rows, n_kv, hd), r(rows, n_kv, hd), r(rows, n_head, hd)
    start = 50
    at = torch.tensor([start], dtype=torch.int32, device=DEV)
    acc = torch.zeros(n_kv, rows, device=DEV)
    args = dict(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=F16, max_rows=rows, block=block)
    a, b = cache.CacheOps(**args), cache.CacheOps(**args)
    bounds = torch.zeros(n_kv, rows // block, 2, hd, dtype=F16, device=DEV)
    b.block_bounds(k, bounds, 0, start)
    k1, v1, q1 = torch.zeros(1, n_kv, hd, device=DEV), torch.zeros(1, n_kv, hd, device=DEV), torch.zeros(1, n_head, hd, device=DEV)
    dense, sparse, rot = (torch.zeros(1, n_head, hd, device=DEV) for _ in range(3))
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a.store(q1, k1, v1, k, v, at, row0_dev=at, q_out=rot)
        a.tree_attention(rot, k, v, n_past_dev=at, acc=acc, out=dense)
    with torch.cuda.graph(g2):
        b.block_attention(rot, k, v, bounds, n_past_dev=at, n_sink=1, n_local=2, n_sel=2, out=sparse)
        b.block_bounds(k, bounds, row1_dev=at)
        at.add_(1)
    weights = torch.zeros(n_kv, rows, dtype=torch.float64)
    for i in range(steps):
        p = start + i
        k1.copy_(kin[p:p + 1]), v1.copy_(vin[p:p + 1]), q1.copy_(qin[p:p + 1])
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert int(at) == p + 1
        if i % 9 == 0 or i == steps - 1:
            want, add = ref.attention(rot, k, v, p)
            assert rel(dense, want) < TOL
            _, seen = ref.blocks(rot, k, p, block, 1, 2, 2)
            assert rel(sparse, ref.attention(rot, k, v, p, past_seen=seen)[0]) < TOL
        weights[:, :p + 1] += ref.attention(rot, k, v, p)[1]
    assert rel(acc, weights) < TOL
    del g1, g2


def test_device_position_is_clamped():
    q, k, v, _ = case(8, 2, 128, F16, 64, 2)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=64, max_tokens=2)
    for value, n in ((-3, 0), (62, 62), (63, 62), (10**9, 62)):
        at = torch.tensor([value], dtype=torch.int32, device=DEV)
        assert rel(ops.tree_attention(q, k, v, n_past_dev=at), ref.attention(q, k, v, n)[0]) < TOL


def test_other_stream():
    q, k, v, _ = case(8, 2, 128, F16, 600, 20)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=600, max_tokens=20)
    want = ops.tree_attention(q, k, v, 580)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(want)
    ops.tree_attention(q, k, v, 580, out=out, stream=s)
    got = ops.tree_attention(q, k, v, 580, stream=s)                     # allocated on the stream of the call
    raw = ops.tree_attention(q, k, v, 580, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(got, want) and torch.equal(raw, want)


def test_long_cache_offsets_pass_32_bits():
    """A cache whose element offsets exceed 2^31."""
    n_kv, hd, rows = 16, 256, 540000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    k = torch.zeros(rows, n_kv, hd, dtype=F16, device=DEV)
    v = torch.zeros_like(k)
    n_past = rows - 1
    assert (rows - 1) * n_kv * hd > 2**31
    q = torch.ones(1, n_kv, hd, device=DEV)
    k[rows - 2, n_kv - 1] = 8.0                       # exp(8 * 256 / 16) dominates
    v[rows - 2, n_kv - 1] = 3.0
    v[0] = 1.0
    ops = cache.CacheOps(n_head=n_kv, n_head_kv=n_kv, head_dim=hd, kv_dtype=F16, max_rows=rows, block=128)
    out = ops.tree_attention(q, k, v, n_past)
    assert rel(out[0, n_kv - 1], torch.full((hd,), 3.0)) < TOL
    assert rel(out[0, 0], torch.full((hd,), 1.0 / rows)) < TOL
    bounds = torch.zeros(n_kv, rows // 128, 2, hd, dtype=F16, device=DEV)
    ops.block_bounds(k, bounds, 0, rows)
    sel = torch.zeros(1, n_kv, 1, dtype=torch.int32, device=DEV)
    out = ops.block_attention(q, k, v, bounds, n_past, n_sink=0, n_local=1, n_sel=1, sel_out=sel)
    assert sel[0, 0, 0] == 0                          # ties: the lowest block
    pos = torch.arange(rows, dtype=torch.int32, device=DEV).repeat(n_kv, 1)
    acc = torch.zeros(n_kv, rows, device=DEV)
    acc[:, rows - 2] = 1.0
    ops.evict(k, v, acc, pos, rows, 10)
    assert (k[0, n_kv - 1] == 0).all() and (k[9, n_kv - 1] == 8).all() and (pos[:, 9] == rows - 2).all()


def test_wrong_tensors_are_refused():
    q, k, v, _ = case(8, 2, 128, F16, 64, 2)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=64, max_tokens=2)
    with pytest.raises(ValueError):
        ops.tree_attention(q.half(), k, v, 3)
    with pytest.raises(ValueError):
        ops.tree_attention(q, k[:60], v[:60], 3)
    with pytest.raises(ValueError):
        ops.tree_attention(q, k, v.transpose(0, 1).contiguous().transpose(0, 1), 3)
    with pytest.raises(ValueError):
        ops.tree_attention(q, k.bfloat16(), v.bfloat16(), 3)
    with pytest.raises(ValueError):
        ops.tree_attention(q, k, v, 3, vis=torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        ops.tree_attention(q.cpu(), k, v, 3)
    with pytest.raises(ValueError):
        ops.block_bounds(k, torch.zeros(2, 4, 2, 128, device=DEV), 0, 64)
    with pytest.raises(HoardError):
        ops.tree_attention(q, k, v, 63)               # the tokens' rows do not fit
    with pytest.raises(HoardError):
        ops.tree_attention(q, k, v, -1)
    with pytest.raises(HoardError):
        ops.tree_attention(torch.cat([q, q]), k, v, 3)        # more tokens than the workspace is for
    with pytest.raises(HoardError):
        ops.tree_attention(q, k, v, 3, acc=torch.zeros(2, 64, device=DEV))    # more than max_acc_tokens
    with pytest.raises(HoardError):
        ops.take(k, v, 0, [1, 1])
    with pytest.raises(HoardError):
        ops.take(k, v, 60, [0, 5])
    with pytest.raises(HoardError):
        ops.evict(k, v, torch.zeros(2, 64, device=DEV), torch.zeros(2, 64, dtype=torch.int32, device=DEV), 10, 11)


def test_expanded_caches_and_wide_integers_are_refused():
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=64, block=16)
    k = torch.zeros(64, 2, 128, dtype=F16, device=DEV)
    q = torch.zeros(1, 8, 128, device=DEV)
    acc, pos = torch.zeros(2, 64, device=DEV), torch.zeros(2, 64, dtype=torch.int32, device=DEV)
    bounds = torch.zeros(2, 4, 2, 128, dtype=F16, device=DEV)
    for flat in (k[:1, :1].expand(64, 2, 128), k[:, :1].expand(64, 2, 128), k[:1].expand(64, 2, 128)):
        with pytest.raises(ValueError):
            ops.tree_attention(q, flat, flat, 3)
        with pytest.raises(ValueError):
            ops.take(flat, flat, 0, [1])
    big = 2**32 + 1
    for call in (lambda: ops.tree_attention(q, k, k, big), lambda: ops.evict(k, k, acc, pos, big, 1),
                 lambda: ops.evict(k, k, acc, pos, 5, 1, recent_from=2**31), lambda: ops.take(k, k, 0, [big]),
                 lambda: ops.take(k, k, big, [1]), lambda: ops.block_bounds(k, bounds, 0, big),
                 lambda: ops.block_attention(q, k, k, bounds, 40, n_sink=1, n_local=1, n_sel=big),
                 lambda: ops.store(q, q[:, :2], q[:, :2], k, k, pos[0, :1], big)):
        with pytest.raises(ValueError):
            call()
