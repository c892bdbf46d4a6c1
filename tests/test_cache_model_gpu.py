"""The cache operators run together in the decode driver (hoard_b200.harness): trees of drafts verified in one forward,
block-sparse and bounded caches, long contexts.

The forms differ from the plain step in the order of the attention's f32 sums, so an activation may round to the other
side of a Q8_K boundary (see test_harness_gpu.py): logits settle ~1e-2 apart, tokens are the same wherever the plain
driver's top two logits are GAP apart, up to the first step where they are not."""
import numpy as np
import pytest
import torch

from hoard_b200 import harness as hx
from tests.moe_fixtures import rel_l2

pytestmark = pytest.mark.gpu

QWEN_S = hx.ModelConfig("qwen3moe", 3, 512, 16, 2, 128, 16, 4, 256, 2048, 1e6, 1e-6, "head", True)
OLMOE_S = hx.ModelConfig("olmoe", 2, 512, 4, 4, 128, 16, 4, 256, 2048, 1e4, 1e-5, "full", False)
HYBRID_S = hx.ModelConfig("qwen3next", 4, 512, 4, 2, 256, 32, 4, 512, 2048, 1e7, 1e-6, "head", True, n_ff_shexp=512,
                          full_attn_interval=4, attn_gate=True, rope_dim=64, ssm_d_state=128, ssm_n_group=2, ssm_dt_rank=4,
                          ssm_d_conv=4)
GAP = 0.05


@pytest.fixture(scope="module")
def weights():
    dev = torch.device("cuda", 0)
    return {id(c): hx.seeded_tensors(c, seed=5, device=dev) for c in (QWEN_S, OLMOE_S, HYBRID_S)}


def make(cfg, weights, **kw):
    return hx.DecodeModel(cfg, weights[id(cfg)], device=0, **kw)


def prompt_of(cfg, n, seed=3):
    return np.random.default_rng(seed).integers(0, cfg.n_vocab, n).tolist()


def plain_run(cfg, weights, prompt, n_gen, **kw):
    m = make(cfg, weights, max_ctx=len(prompt) + n_gen + 40, **kw)
    logits = torch.empty(n_gen, cfg.n_vocab, device="cuda:0")
    tokens = m.generate(prompt, n_gen, logits_out=logits)
    m.close()
    top = torch.topk(logits, 2, 1).values
    return tokens, (top[:, 0] - top[:, 1]).tolist(), logits


def same_up_to_a_near_tie(got, want, gaps):
    for i, (a, b) in enumerate(zip(got, want)):
        if a != b:
            assert gaps[i] < GAP, (i, a, b, gaps[i])
            return i
    return len(want)


@pytest.mark.parametrize("cfg", [QWEN_S, OLMOE_S])
@pytest.mark.parametrize("kv", [torch.float16, torch.bfloat16])
def test_forward_tree_matches_its_paths(cfg, kv, weights):
    prompt = prompt_of(cfg, 70)
    m = make(cfg, weights, max_ctx=200, kv_dtype=kv, max_batch=24)
    m.generate(prompt, 1)
    tokens = prompt_of(cfg, 21, seed=9)
    parents = [-1, -1, 0, 0, 1, 2, 2, 5, 5, 7, 4, 10, 11, -1, 13, 14, 15, 16, 17, 18, 19]
    out = m.forward_tree(tokens, parents, len(prompt))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    again = m.forward_tree(tokens, parents, len(prompt), stream=side)
    side.synchronize()
    assert torch.equal(again, out)
    for leaf in (3, 6, 8, 9, 12, 20):
        path = []
        i = leaf
        while i >= 0:
            path.insert(0, i)
            i = parents[i]
        chain = m.forward_batch([tokens[i] for i in path], len(prompt))
        rel = [rel_l2(out[i].cpu().numpy(), chain[j].cpu().numpy()) for j, i in enumerate(path)]
        assert np.median(rel) < 2e-2 and max(rel) < 5e-2, (leaf, rel)
    # the accepted path's rows become the chain's rows
    m.forward_tree(tokens, parents, len(prompt))
    path = [0, 2, 5, 7, 9]
    m.accept(len(prompt), path)
    kept = m.kc[:, 70:75].clone()
    m.forward_batch([tokens[i] for i in path], 70)
    assert rel_l2(kept.float().cpu().numpy(), m.kc[:, 70:75].float().cpu().numpy()) < 5e-2
    assert torch.equal(kept[0], m.kc[0, 70:75])       # the first layer's keys do not depend on attention
    with pytest.raises(ValueError):
        m.forward_tree(tokens, parents[:-1], 70)
    with pytest.raises(ValueError):
        m.forward_tree([1] * 25, [-1] * 25, 70)
    with pytest.raises(ValueError):
        m.forward_tree(tokens, parents, 190)
    m.close()


@pytest.mark.parametrize("depth,width", [(1, 1), (3, 2), (4, 4)])
def test_tree_generate_is_lossless(depth, width, weights):
    cfg, n_gen = QWEN_S, 40
    prompt = prompt_of(cfg, 33)
    want, gaps, _ = plain_run(cfg, weights, prompt, n_gen)
    m = make(cfg, weights, max_ctx=160)
    got, stats = m.tree_generate(prompt, n_gen, depth=depth, width=width)
    assert len(got) == n_gen and stats["proposed"] == stats["rounds"] * depth * width
    same_up_to_a_near_tie(got, want, gaps)
    with pytest.raises(ValueError):
        m.tree_generate(prompt, 4, depth=9, width=2)          # 18 drafts, max_batch 16
    m.close()


@pytest.mark.parametrize("cfg", [QWEN_S, HYBRID_S])
def test_every_block_chosen_is_the_plain_attention(cfg, weights):
    n_gen = 40
    prompt = prompt_of(cfg, 90)
    want, gaps, _ = plain_run(cfg, weights, prompt, n_gen)
    m = make(cfg, weights, max_ctx=160, blocks=hx.BlockChoice(block=16, n_sink=1, n_local=1, n_sel=100))
    same_up_to_a_near_tie(m.generate(prompt, n_gen), want, gaps)
    same_up_to_a_near_tie(m.generate_graphed(prompt, n_gen), want, gaps)
    if cfg is QWEN_S:
        got, _ = m.tree_generate(prompt, 20, depth=3, width=3)
        same_up_to_a_near_tie(got, want[:20], gaps)
    m.close()


@pytest.mark.parametrize("cfg", [QWEN_S, HYBRID_S])
def test_few_blocks(cfg, weights):
    """The graph's position in device memory chooses the blocks that the eager driver does; bounds are those of the cache."""
    prompt, n_gen, blk = prompt_of(cfg, 150), 30, hx.BlockChoice(block=16, n_sink=1, n_local=2, n_sel=3)
    m = make(cfg, weights, max_ctx=256, blocks=blk)
    logits = torch.empty(n_gen, cfg.n_vocab, device="cuda:0")
    got = m.generate(prompt, n_gen, logits_out=logits)
    top = torch.topk(logits, 2, 1).values
    done = (150 + n_gen - 1) // 16
    for i in range(len(m.kv_index)):
        kb = m._heads(m.kc[i])[:done * 16].view(done, 16, cfg.n_head_kv, cfg.head_dim)
        assert torch.equal(m.bounds[i][:, :done, 0].transpose(0, 1), kb.amin(1))
        assert torch.equal(m.bounds[i][:, :done, 1].transpose(0, 1), kb.amax(1))
    same_up_to_a_near_tie(m.generate_graphed(prompt, n_gen), got, (top[:, 0] - top[:, 1]).tolist())
    m.close()


@pytest.mark.parametrize("cfg", [QWEN_S, HYBRID_S])
def test_budget_that_holds_everything_is_the_plain_attention(cfg, weights):
    n_gen = 40
    prompt = prompt_of(cfg, 60)
    want, gaps, _ = plain_run(cfg, weights, prompt, n_gen)
    m = make(cfg, weights, max_ctx=160, budget=hx.CacheBudget(n_keep=140, n_slack=20))
    same_up_to_a_near_tie(m.generate(prompt, n_gen), want, gaps)
    # every token's weights add up to one per head
    n = len(prompt) + n_gen - 1
    total = m.kv_acc[:, :, :n].sum(2).cpu()
    assert torch.allclose(total, torch.full_like(total, float(n * cfg.n_head // cfg.n_head_kv)), rtol=1e-4)
    same_up_to_a_near_tie(m.generate_graphed(prompt, n_gen), want, gaps)
    m.close()


@pytest.mark.parametrize("cfg", [QWEN_S, HYBRID_S])
def test_budget_evicts(cfg, weights):
    prompt, n_gen = prompt_of(cfg, 100), 60
    b = hx.CacheBudget(n_keep=48, n_slack=16, n_sink=3, n_recent=20)
    m = make(cfg, weights, max_ctx=200, budget=b)
    logits = torch.empty(n_gen, cfg.n_vocab, device="cuda:0")
    got = m.generate(prompt, n_gen, logits_out=logits)
    n = 100 + n_gen - 1                                 # tokens stored
    assert m.kc.shape[1] == 64 and m.n_rows == n - 16 * ((n - 64 + 15) // 16)
    last = n - m.n_rows + b.n_keep                      # position of the first token after the last eviction
    for i in range(len(m.kv_index)):
        pos = m.kv_pos[i][:, :m.n_rows].cpu()
        for h in range(cfg.n_head_kv):
            held = pos[h].tolist()
            assert len(set(held)) == m.n_rows and max(held) == n - 1
            assert set(range(b.n_sink)) <= set(held) and set(range(last - b.n_recent, n)) <= set(held)
    top = torch.topk(logits, 2, 1).values
    same_up_to_a_near_tie(m.generate_graphed(prompt, n_gen), got, (top[:, 0] - top[:, 1]).tolist())
    for call in (lambda: m.forward_batch([1, 2], 10), lambda: m.speculative_generate(prompt, 4),
                 lambda: m.tree_generate(prompt, 4), lambda: m.forward_tree([1], [-1], 10)):
        with pytest.raises(ValueError):
            call()
    m.close()


def test_context_beyond_shared_memory(weights):
    """A cache too long for the one-CTA attention's scores."""
    cfg, n_gen = QWEN_S, 12
    prompt = prompt_of(cfg, 40)
    want, gaps, _ = plain_run(cfg, weights, prompt, n_gen)
    m = make(cfg, weights, max_ctx=60000)
    same_up_to_a_near_tie(m.generate(prompt, n_gen), want, gaps)
    same_up_to_a_near_tie(m.generate_graphed(prompt, n_gen), want, gaps)
    m.close()


def test_wrong_settings_are_refused(weights):
    for bad in (dict(max_batch=0), dict(max_batch=65), dict(blocks=hx.BlockChoice(), budget=hx.CacheBudget(64)),
                dict(budget=hx.CacheBudget(n_keep=100, n_sink=50, n_recent=50)), dict(budget=hx.CacheBudget(64, n_slack=0, n_recent=8)),
                dict(kv_dtype=torch.float32), dict(blocks=hx.BlockChoice(block=128))):
        with pytest.raises(ValueError):
            make(OLMOE_S, weights, max_ctx=64, **bad)
    m = make(HYBRID_S, weights, max_ctx=64)
    with pytest.raises(ValueError):
        m.forward_tree([1], [-1], 3)
    with pytest.raises(ValueError):
        m.tree_generate([1, 2, 3], 4)
    m.close()
    m = make(OLMOE_S, weights, max_ctx=64)
    with pytest.raises(ValueError):
        m.accept(3, [0])                                 # no tree yet
    m.forward_tree([1, 2], [-1, 0], 3)
    with pytest.raises(ValueError):
        m.accept(3, [0, 2])
    m.accept(3, [])
    m.close()
