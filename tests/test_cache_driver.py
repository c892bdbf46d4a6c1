"""What the decode driver refuses of the cache operators, on the CPU: the checks come before anything is launched."""
import types

import pytest

from hoard_b200 import harness as hx


def driver(**kw):
    """A DecodeModel with its settings alone."""
    m = hx.DecodeModel.__new__(hx.DecodeModel)
    m.cfg = types.SimpleNamespace(n_expert_used=4, full_attn_interval=0)
    m.budget, m.blocks, m.max_ctx, m.max_batch = None, None, 160, 16
    for k, v in kw.items():
        setattr(m, k, v)
    return m


def test_blocks_that_are_left_out():
    b = hx.BlockChoice(block=16, n_sink=1, n_local=2, n_sel=3)
    assert not b.leaves_out(0) and not b.leaves_out(96) and b.leaves_out(97)
    assert not hx.BlockChoice(block=16, n_sink=1, n_local=1, n_sel=100).leaves_out(160)


@pytest.mark.parametrize("blocks", [hx.BlockChoice(block=16, n_sink=1, n_local=1, n_sel=4), hx.BlockChoice(block=16, n_sink=0, n_local=1, n_sel=0)])
def test_tree_generate_refuses_blocks_that_are_left_out(blocks):
    with pytest.raises(ValueError, match="blocks"):
        driver(blocks=blocks).tree_generate(list(range(90)), 4, depth=3, width=2)


def test_positions_of_the_one_cta_attention():
    """One position more than plain_attention_rows says is refused (before anything is launched)."""
    one = 4096
    for hd in (8, 16, 64, 128, 256, 4, 2):
        n = hx.plain_attention_rows(hd)
        assert n > 40000 and hx._hx().hoard_hx_attention(one, one, one, 4, 2, hd, n + 1, 0.1, one, 1, None) == -1
    for hd in (0, 96, 80, 512):
        assert hx.plain_attention_rows(hd) == 0
