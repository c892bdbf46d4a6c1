"""The cache operators at the ends of the number range: whatever is finite in plain f32 stays finite, in every kernel of the
dense attention. Definitions and tolerances as in test_cache_gpu.py; inputs here are such that the definition's weights are
known whatever the scores' last bits are (keys of one level score alike to the bit; levels lie far apart), or
that the range is extreme in q and k and ordinary in the scores."""
import pytest
import torch

from hoard_b200 import cache
from tests import cache_ref as ref
from tests.cache_forms import SHAPES, attention64, kernel_of
from tests.test_cache_gpu import BF16, DEV, F16, TOL, case, rel, tree

pytestmark = pytest.mark.gpu
shapes = pytest.mark.parametrize("s", SHAPES, ids=lambda s: s["kernel"].replace(", ", "_").replace(" ", "_"))


def levels(n_head, n_kv, hd, m, n_past, kt, sign, low=23, high=34):
    """Keys of nine levels 2^15 (1 - l / 16), queries that bring the largest score of row i to sign * 2^low .. 2^high in units
    of log2: two levels are at least 2^(low - 4) apart there, far above a step of f32 (2^(low - 23))."""
    g = torch.Generator(device=DEV).manual_seed(m)
    n = n_past + m
    level = torch.randint(0, 9, (n, n_kv), generator=g, device=DEV)
    level[0] = 0 if sign > 0 else 8
    k = (2.0**15 * (1 - level / 16.0))[..., None].expand(n, n_kv, hd).contiguous().to(kt)
    top = 2.0 ** torch.linspace(low, high, m * n_head, device=DEV, dtype=torch.float64)
    q = sign * (top * 0.6931471805599453 / (hd**0.5 * 2.0**15)).float().view(m, n_head, 1).expand(m, n_head, hd).contiguous()
    v = torch.randn(n, n_kv, hd, generator=g, device=DEV).to(kt)
    return q, k, v


@shapes
@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(s, kt, sign):
    assert kernel_of(s, kt) == s["kernel"]
    q, k, v = levels(s["n_head"], s["n_kv"], s["hd"], s["m"], s["n_past"], kt, sign)
    ops = cache.CacheOps(n_head=s["n_head"], n_head_kv=s["n_kv"], head_dim=s["hd"], kv_dtype=kt, max_rows=s["n_past"] + s["m"],
                         max_tokens=s["m"])
    vis, _ = tree(s["m"], 2)
    want = attention64(q, k, v, s["n_past"], vis)
    out = ops.tree_attention(q, k, v, s["n_past"], vis=vis)
    assert torch.isfinite(out).all() and rel(out, want) < TOL


@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("n_head,n_kv,hd,m,n_past", [(8, 2, 128, 1, 300), (8, 2, 128, 2, 40), (8, 2, 64, 1, 3000), (16, 2, 256, 3, 700)])
def test_large_scores_accumulated(n_head, n_kv, hd, m, n_past, kt, sign):
    q, k, v = levels(n_head, n_kv, hd, m, n_past, kt, sign)
    n = n_past + m
    ops = cache.CacheOps(n_head=n_head, n_head_kv=n_kv, head_dim=hd, kv_dtype=kt, max_rows=n, max_tokens=m, max_acc_tokens=m)
    acc = torch.zeros(n_kv, n, device=DEV)
    out = ops.tree_attention(q, k, v, n_past, acc=acc)
    want, add = ref.attention(q, k, v, n_past)
    assert rel(out, want) < TOL and rel(acc, add) < TOL


@shapes
@pytest.mark.parametrize("kt", [F16, BF16])
@pytest.mark.parametrize("size", [3.4028234663852886e38, 3.401e38])
def test_queries_of_the_largest_float(s, kt, size):
    """Up to the largest float itself a query is finite. Its other dims are 0 and keys have levels there, so that equal scores
    share the weight."""
    m, n_past, n = s["m"], s["n_past"], s["n_past"] + s["m"]
    assert kernel_of(s, kt) == s["kernel"]
    _, k, v, r = case(s["n_head"], s["n_kv"], s["hd"], kt, n, m)
    k[:, :, 0] = torch.randint(1, 6, (n, s["n_kv"]), device=DEV).to(kt) * 2.0**-24
    q = torch.zeros(m, s["n_head"], s["hd"], device=DEV)
    q[:, :, 0] = size * torch.sign(r(m, s["n_head"]))
    ops = cache.CacheOps(n_head=s["n_head"], n_head_kv=s["n_kv"], head_dim=s["hd"], kv_dtype=kt, max_rows=n, max_tokens=m)
    out = ops.tree_attention(q, k, v, n_past)
    assert rel(out, attention64(q, k, v, n_past)) < TOL


@shapes
@pytest.mark.parametrize("down,up", [(-100, 127), (-60, 127), (-5, 127), (-140, 127), (100, -100), (124, -120)])
def test_small_queries_beside_large_keys(s, down, up):
    """bf16 has f32's range: scores of ordinary size from queries and keys of opposite extremes (q of 2^-140 is subnormal in f32)."""
    assert kernel_of(s, BF16) == s["kernel"]
    m, n_past, n = s["m"], s["n_past"], s["n_past"] + s["m"]
    q, k, v, _ = case(s["n_head"], s["n_kv"], s["hd"], BF16, n, m)
    q, k = q * 2.0**down, (k.float() * 2.0**up).clamp(-3.3e38, 3.3e38).to(BF16)
    scale = 2.0 ** -(down + up) / s["hd"] ** 0.5
    ops = cache.CacheOps(n_head=s["n_head"], n_head_kv=s["n_kv"], head_dim=s["hd"], kv_dtype=BF16, max_rows=n, max_tokens=m,
                         scale=scale)
    assert rel(ops.tree_attention(q, k, v, n_past), attention64(q, k, v, n_past, scale=scale)) < TOL


@shapes
@pytest.mark.parametrize("kt", [F16, BF16])
def test_scores_that_vanish(s, kt):
    """A scale and queries so small that their product is 0 in f32: equal weights for the rows that are seen, none for the others."""
    assert kernel_of(s, kt) == s["kernel"]
    m, n_past, n = s["m"], s["n_past"], s["n_past"] + s["m"]
    q, k, v, _ = case(s["n_head"], s["n_kv"], s["hd"], kt, n, m)
    ops = cache.CacheOps(n_head=s["n_head"], n_head_kv=s["n_kv"], head_dim=s["hd"], kv_dtype=kt, max_rows=n, max_tokens=m, scale=1e-30)
    vis, _ = tree(m, 6)
    q = q * (1e-30 if kt is F16 else 1e-37)
    assert rel(ops.tree_attention(q, k, v, n_past, vis=vis), attention64(q, k, v, n_past, vis, scale=1e-30)) < TOL
