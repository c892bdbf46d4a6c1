"""The decode driver's use of the cache operators, beside test_cache_model_gpu.py: what a tree attends where blocks are left out."""
import pytest
import torch

from hoard_b200 import harness as hx
from tests import cache_ref as ref
from tests.test_cache_gpu import TOL, rel
from tests.test_cache_model_gpu import OLMOE_S, QWEN_S, prompt_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights():
    dev = torch.device("cuda", 0)
    return {c.arch: hx.seeded_tensors(c, seed=5, device=dev) for c in (QWEN_S, OLMOE_S)}


def make(cfg, weights, **kw):
    return hx.DecodeModel(cfg, weights[cfg.arch], device=0, **kw)


@pytest.mark.parametrize("cfg", [QWEN_S, OLMOE_S])
def test_forward_tree_over_few_blocks(cfg, weights):
    """Blocks are chosen for the past before the tree, whatever the tokens' depths; the drafts cross the end of a block."""
    base, prompt = 47, prompt_of(cfg, 60)
    m = make(cfg, weights, max_ctx=128, blocks=hx.BlockChoice(block=16, n_sink=0, n_local=1, n_sel=1))
    m.generate(prompt[:base], 1)
    calls = []
    m.forward_tree(prompt[:1], [-1], base)             # makes the tree's operators
    run = m._tree_ops.block_attention

    def recorded(q, k, v, bounds, n_past, **kw):
        out = run(q, k, v, bounds, n_past, **kw)
        calls.append((q.clone(), k.clone(), v.clone(), n_past, kw["vis"].clone(), out.clone()))
        return out

    m._tree_ops.block_attention = recorded
    parents = [-1, 0, 1, 2, 0, 4, -1]
    m.forward_tree(prompt[base:base + 7], parents, base)
    assert len(calls) == cfg.n_layer
    for q, k, v, n_past, vis, out in calls:
        assert n_past == base
        chosen, seen = ref.blocks(q, k, base, 16, 0, 1, 1)
        assert all(len(c) == 1 and c[0] in (0, 1) for t in chosen for c in t) and not seen.all()
        assert rel(out, ref.attention(q, k, v, base, vis, past_seen=seen)[0]) < TOL
    m.close()
