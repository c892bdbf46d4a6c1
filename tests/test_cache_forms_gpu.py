"""Every kernel of the cache operators on the calls where it can go wrong: the dense attention's mma form, its tensor-core
form with and without splits, the block choice's three forms. Definitions and tolerances as in test_cache_gpu.py."""
import pytest
import torch

from hoard_b200 import cache
from tests import cache_ref as ref
from tests.cache_forms import CHOOSE, SHAPES, attention64, choose_form, kernel_of
from tests.test_cache_gpu import BF16, DEV, F16, TOL, case, rel, tree

pytestmark = pytest.mark.gpu
shapes = pytest.mark.parametrize("s", SHAPES, ids=lambda s: s["kernel"].replace(", ", "_").replace(" ", "_"))
both = pytest.mark.parametrize("kt", [F16, BF16])


def setup(s, kt, extra=0, **kw):
    assert kernel_of(s, kt) == s["kernel"]
    n = s["n_past"] + s["m"]
    q, k, v, r = case(s["n_head"], s["n_kv"], s["hd"], kt, n + extra, s["m"])
    ops = cache.CacheOps(n_head=s["n_head"], n_head_kv=s["n_kv"], head_dim=s["hd"], kv_dtype=kt, max_rows=n + extra,
                         max_tokens=s["m"], **kw)
    return q, k, v, r, ops


@shapes
@both
@pytest.mark.parametrize("pad", [0, 3])
def test_strides_and_gate(s, kt, pad):
    """q and gate inside wider rows (16-byte aligned heads, and not), a cache laid out [head][row][dim], an output that is given."""
    q, k, v, r, ops = setup(s, kt)
    hd, n_past = s["hd"], s["n_past"]
    vis, _ = tree(s["m"], 5)
    fused = r(s["m"], s["n_head"], 2 * hd + pad)
    fused[..., :hd] = q
    qs, gate = fused[..., :hd], fused[..., hd:2 * hd]
    kh, vh = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    out = torch.full((s["m"], s["n_head"], hd), float("nan"), device=DEV)
    ops.tree_attention(qs, kh, vh, n_past, vis=vis, gate=gate, out=out)
    want = attention64(q, k, v, n_past, vis, gate)
    assert rel(out, want) < TOL
    assert torch.equal(ops.tree_attention(qs, k, v, n_past, vis=vis, gate=gate), out)
    chain = ops.tree_attention(qs, k, v, n_past)
    assert rel(chain, attention64(q, k, v, n_past)) < TOL


@shapes
@both
def test_masked_rows_may_hold_anything(s, kt):
    q, k, v, _, ops = setup(s, kt)
    m, n_past = s["m"], s["n_past"]
    vis, _ = tree(m, 3)
    clean = ops.tree_attention(q, k, v, n_past, vis=vis)
    for bad in (m - 2, 1):
        sees = ref.visibility(vis, m)[:, bad].to(DEV)
        assert sees.any() and not sees.all()
        for value in (float("inf"), float("-inf"), float("nan")):
            k2, v2 = k.clone(), v.clone()
            v2[n_past + bad, :, ::2] = value
            out = ops.tree_attention(q, k, v2, n_past, vis=vis)
            assert rel(out[~sees], clean[~sees]) < TOL and not torch.isfinite(out[sees][..., ::2]).any()
            assert rel(out[sees][..., 1::2], clean[sees][..., 1::2]) < TOL
            if value == value:
                assert (out[sees][..., ::2] == value).all()
            k2[n_past + bad] = value
            out = ops.tree_attention(q, k2, v2, n_past, vis=vis)
            assert rel(out[~sees], clean[~sees]) < TOL


@shapes
@both
def test_nan_query_stays_in_its_row(s, kt):
    q, k, v, _, ops = setup(s, kt)
    clean = ops.tree_attention(q, k, v, s["n_past"])
    for value in (float("nan"), float("inf")):
        q2 = q.clone()
        q2[1, 5, 7] = value
        out = ops.tree_attention(q2, k, v, s["n_past"])
        assert torch.isnan(out[1, 5]).all()
        out[1, 5] = clean[1, 5]
        assert torch.equal(out, clean)


@shapes
@both
def test_visibility_bits_beyond_the_tokens(s, kt):
    q, k, v, _, ops = setup(s, kt, extra=64)
    m, n = s["m"], s["n_past"] + s["m"]
    k[n:], v[n:] = float("nan"), float("nan")
    every = torch.full((m,), -1, dtype=torch.int64, device=DEV)
    just = torch.full((m,), (1 << m) - 1, dtype=torch.int64, device=DEV)
    out = ops.tree_attention(q, k, v, s["n_past"], vis=every)
    assert torch.equal(out, ops.tree_attention(q, k, v, s["n_past"], vis=just))
    assert rel(out, attention64(q, k, v, s["n_past"], just)) < TOL


@shapes
@both
def test_head_major_queries_and_output_in_place(s, kt):
    q, k, v, r, ops = setup(s, kt)
    gate = r(s["n_head"], s["m"], s["hd"]).transpose(0, 1)
    want = ops.tree_attention(q, k, v, s["n_past"], gate=gate)
    assert rel(want, attention64(q, k, v, s["n_past"], None, gate)) < TOL
    major = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.tree_attention(major, k, v, s["n_past"], gate=gate), want)
    x = q.clone()
    assert ops.tree_attention(x, k, v, s["n_past"], gate=gate, out=x) is x and torch.equal(x, want)


@shapes
@both
def test_other_stream(s, kt):
    q, k, v, _, ops = setup(s, kt)
    want = ops.tree_attention(q, k, v, s["n_past"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(want)
    ops.tree_attention(q, k, v, s["n_past"], out=out, stream=side)
    raw = ops.tree_attention(q, k, v, s["n_past"], stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(raw, want)


@shapes
@both
def test_position_in_device_memory(s, kt):
    """One captured call at positions from none to the last."""
    q, k, v, r, ops = setup(s, kt)
    gate, at = r(s["m"], s["n_head"], s["hd"]), torch.zeros(1, dtype=torch.int32, device=DEV)
    vis, _ = tree(s["m"], 8)
    out = torch.zeros(s["m"], s["n_head"], s["hd"], device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attention(q, k, v, vis=vis, gate=gate, n_past_dev=at, out=out)
    for n in (0, 1, 63, 64, 65, s["n_past"] // 2, s["n_past"]):
        at.fill_(n)
        graph.replay()
        assert rel(out, attention64(q, k, v, n, vis, gate)) < TOL
    del graph


# candidates, KV heads x tokens, layout, form. Keys of a problem: in one CTA of 512 threads in rounds of 2048, in a cluster
# an eighth each
@pytest.mark.parametrize("n_cand,n_head,n_kv,hd,m,block,kt,form", [
    (1500, 2, 1, 64, 1, 16, F16, CHOOSE[1]), (4000, 8, 2, 128, 1, 16, BF16, CHOOSE[1]), (8192, 12, 1, 40, 1, 16, F16, CHOOSE[1]),
    (2500, 4, 2, 256, 2, 16, F16, CHOOSE[1]), (3001, 20, 1, 32, 3, 16, BF16, CHOOSE[1]),
    (3000, 40, 20, 16, 1, 16, F16, CHOOSE[0]), (6001, 20, 10, 32, 2, 16, BF16, CHOOSE[0]), (2049, 24, 2, 136, 10, 16, F16, CHOOSE[0]),
    (8193, 4, 2, 24, 1, 16, F16, CHOOSE[2])])
@pytest.mark.parametrize("n_sel", [1, 77, 1400])
def test_block_choice_of_each_form(n_cand, n_head, n_kv, hd, m, block, kt, form, n_sel):
    assert choose_form(n_cand, n_kv * m) == form
    n_sink, n_local = 2, 3
    n_past = (n_cand + n_sink + n_local) * block - 5
    q, k, v, _ = case(n_head, n_kv, hd, kt, n_past + m, m, seed=n_cand + n_sel)
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=n_past + m, max_tokens=m, block=block)
    bounds = ops.block_bounds(k, torch.zeros(n_kv, (n_past + m) // block, 2, hd, dtype=kt, device=DEV), 0, n_past)
    sel = torch.full((m, n_kv, n_sel), -7, dtype=torch.int32, device=DEV)
    out = ops.block_attention(q, k, v, bounds, n_past, n_sink=n_sink, n_local=n_local, n_sel=n_sel, sel_out=sel)
    chosen, seen = ref.blocks(q, k, n_past, block, n_sink, n_local, n_sel)
    assert sel.tolist() == chosen
    some = range(0, n_head, max(1, n_head // 4))          # the attention over the list, for some heads
    g = n_head // n_kv
    for h in some:
        want, _ = ref.attention(q[:, h:h + 1], k[:, h // g:h // g + 1], v[:, h // g:h // g + 1], n_past, past_seen=seen[:, h // g:h // g + 1])
        assert rel(out[:, h:h + 1], want) < TOL


@pytest.mark.parametrize("given", ["stream", "handle", "current"])
def test_workspace_of_a_running_call_is_not_given_away(given):
    """A CacheOps that is dropped while its call on another stream waits: its workspace is nobody else's before that is done."""
    q, k, v, _ = case(8, 2, 128, F16, 600, 20)
    ops = cache.CacheOps(n_head=8, n_head_kv=2, head_dim=128, kv_dtype=F16, max_rows=600, max_tokens=20)
    want = ops.tree_attention(q, k, v, 580)
    out = torch.empty_like(want)
    at, size = ops._ws.data_ptr(), ops._ws.numel()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)                   # about 0.2 s, after which the call runs
        if given == "current":
            ops.tree_attention(q, k, v, 580, out=out)
    if given != "current":
        ops.tree_attention(q, k, v, 580, out=out, stream=side if given == "stream" else side.cuda_stream)
    del ops
    held = [torch.empty(size, dtype=torch.uint8, device=DEV) for _ in range(3)]
    busy = not side.query()
    assert busy and at not in [x.data_ptr() for x in held]
    side.synchronize()
    assert torch.equal(out, want)
    del held
