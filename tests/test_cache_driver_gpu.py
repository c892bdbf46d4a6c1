"""The decode driver's use of the cache operators, beside test_cache_model_gpu.py: what a tree attends where blocks are left out,
trees whose drafts are accepted, generated tokens against the plain model's logits after any near tie."""
import dataclasses

import pytest
import torch

from hoard_b200 import harness as hx
from tests import cache_ref as ref
from tests.test_cache_gpu import TOL, rel
from tests.test_cache_model_gpu import GAP, OLMOE_S, QWEN_S, prompt_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights():
    dev = torch.device("cuda", 0)
    return {c.arch: hx.seeded_tensors(c, seed=5, device=dev) for c in (QWEN_S, OLMOE_S)}


def make(cfg, weights, **kw):
    return hx.DecodeModel(cfg, weights[cfg.arch], device=0, **kw)


def assert_greedy(cfg, weights, prompt, tokens, **kw):
    """Every generated token is the plain model's best after those before it, or within GAP of it."""
    m = make(cfg, weights, max_ctx=len(prompt) + len(tokens) + 8, **kw)
    logits = m.score(prompt + tokens, len(prompt))
    m.close()
    got = logits.gather(1, torch.tensor(tokens, device=logits.device)[:, None])[:, 0]
    assert float((logits.amax(1) - got).max()) < GAP


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


@pytest.mark.parametrize("cfg", [QWEN_S, OLMOE_S])
@pytest.mark.parametrize("depth,width", [(4, 3), (1, 8)])
def test_trees_of_the_model_itself_are_accepted(cfg, depth, width, weights):
    """With one expert the draft is the full model: its best path is accepted, and the rows that are taken over serve every
    later round."""
    cfg, n_gen = dataclasses.replace(cfg, n_expert_used=1), 40
    prompt = prompt_of(cfg, 33)
    m = make(cfg, weights, max_ctx=160)
    got, stats = m.tree_generate(prompt, n_gen, depth=depth, width=width)
    m.close()
    assert len(got) == n_gen and stats["accepted"] >= 0.8 * depth * stats["rounds"]
    assert stats["rounds"] < n_gen / (1 + 0.7 * depth) + 1
    assert_greedy(cfg, weights, prompt, got)


@pytest.mark.parametrize("cfg", [QWEN_S, OLMOE_S])
def test_tree_generate_is_greedy(cfg, weights):
    prompt, n_gen = prompt_of(cfg, 33), 40
    for kw in (dict(), dict(blocks=hx.BlockChoice(block=16, n_sink=1, n_local=1, n_sel=20))):
        m = make(cfg, weights, max_ctx=160, **kw)
        got, _ = m.tree_generate(prompt, n_gen, depth=3, width=4)
        m.close()
        assert_greedy(cfg, weights, prompt, got)


def test_long_contexts_keep_the_plain_attention_where_it_runs(weights):
    """The same bits whatever max_ctx is: eager steps up to the positions that the one-CTA attention takes, captured ones up to
    contexts of as many."""
    cfg, n_gen = QWEN_S, 12
    prompt = prompt_of(cfg, 40)
    runs = []
    for max_ctx in (60, 46976, 60000):
        m = make(cfg, weights, max_ctx=max_ctx)
        assert m.plain_rows == 46976
        logits = torch.empty(n_gen, cfg.n_vocab, device="cuda:0")
        tokens = m.generate(prompt, n_gen, logits_out=logits)
        graphed = m.generate_graphed(prompt, n_gen)
        runs.append((tokens, logits, graphed, m.logits.clone()))
        m.close()
    for tokens, logits, graphed, last in runs[1:]:
        assert tokens == runs[0][0] and torch.equal(logits, runs[0][1])
    assert runs[1][2] == runs[0][2] and torch.equal(runs[1][3], runs[0][3])
    assert_greedy(cfg, weights, prompt, runs[2][2])


def test_the_step_where_the_plain_attention_ends(weights):
    cfg = QWEN_S
    m = make(cfg, weights, max_ctx=47100)
    m.kc.normal_(std=0.5), m.vc.normal_(std=0.5)
    m.seq.fill_(11)
    for pos in (m.plain_rows - 1, m.plain_rows, 47099):
        m.step(pos, m.scratch_tok)
        step = m.logits.clone()
        tree = m.forward_tree([11], [-1], pos)[0]
        assert torch.isfinite(step).all() and rel(tree, step) < 2e-2, pos
    m.close()


def test_layouts_that_only_the_plain_attention_takes():
    """More than 64 query heads per KV head: a long context is served up to the positions of the one-CTA attention."""
    cfg = hx.ModelConfig("qwen3moe", 1, 512, 256, 2, 8, 16, 4, 256, 2048, 1e6, 1e-6, "head", True)
    tensors, prompt, runs = hx.seeded_tensors(cfg, seed=5, device=torch.device("cuda", 0)), prompt_of(cfg, 20), []
    for max_ctx in (40, 60000):
        m = hx.DecodeModel(cfg, tensors, device=0, max_ctx=max_ctx)
        assert m.ops is None
        logits = torch.empty(8, cfg.n_vocab, device="cuda:0")
        runs.append((m.generate(prompt, 8, logits_out=logits), logits))
        if max_ctx == 60000:
            with pytest.raises(hx.HoardError):
                m.step(m.plain_rows, m.scratch_tok)
        m.close()
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1])
    with pytest.raises(hx.HoardError):
        hx.DecodeModel(cfg, tensors, device=0, max_ctx=200, budget=hx.CacheBudget(64, n_recent=8))


def test_trees_in_a_context_shorter_than_the_largest_batch(weights):
    cfg = OLMOE_S
    m = make(cfg, weights, max_ctx=8)
    prompt = prompt_of(cfg, 3)
    m.generate(prompt, 1)
    out = m.forward_tree([5, 6, 7, 8, 9], [-1, 0, 0, 2, -1], 3)
    chain = m.forward_batch([5, 7, 8], 3)
    for i, j in ((0, 0), (2, 1), (3, 2)):
        assert rel(out[i], chain[j]) < 5e-2
    with pytest.raises(ValueError):
        m.forward_tree([1] * 6, [-1] * 6, 3)
    m.close()


@pytest.mark.parametrize("hd", [128, 256])
def test_batches_of_a_gated_attention(hd):
    """Layers with an output gate and no delta-net between them: a token's q row in a batch holds its gate, and a tree goes
    through the operators with it."""
    cfg = dataclasses.replace(QWEN_S, n_head=8, head_dim=hd, attn_gate=True, rope_dim=64)
    m = hx.DecodeModel(cfg, hx.seeded_tensors(cfg, seed=5, device=torch.device("cuda", 0)), device=0, max_ctx=80, max_batch=6)
    prompt = prompt_of(cfg, 30)
    tokens = prompt_of(cfg, 6, seed=8)
    m.generate(prompt, 1)
    assert m._q_view(m.q).shape == m._gate_view(m.q).shape == (1, 8, hd)
    out = m.forward_batch(tokens, 30)
    steps = m.score(prompt + tokens + [0], 31)
    assert all(rel(out[i], steps[i]) < 5e-2 for i in range(6))
    m.generate(prompt, 1)
    tree = m.forward_tree(tokens, [-1, 0, 1, 2, 3, 4], 30)
    assert all(rel(tree[i], out[i]) < 5e-2 for i in range(6))
    m.close()
