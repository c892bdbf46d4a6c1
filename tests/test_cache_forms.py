"""The rules by which the cache operators choose a kernel, asked on the CPU: the shapes of the GPU tests reach the kernels they
are for, and so do sizes that the benchmark and the driver have."""
import pytest
import torch

from tests.cache_forms import CHOOSE, MMA, SHAPES, TC, attention_form, choose_form, kernel_of

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("kt", [F16, BF16])
def test_shapes_reach_their_kernels(kt):
    assert [kernel_of(s, kt) for s in SHAPES] == [s["kernel"] for s in SHAPES]


def test_attention_forms():
    assert attention_form(32, 4, 128, F16, 42, 5, 37)[0] == MMA and attention_form(32, 4, 128, F16, 131072, 64, 131008)[0] == TC
    for acc in (False, True):                          # weights are accumulated beside the mma form alone
        assert attention_form(32, 4, 128, BF16, 4111, 16, 4095, acc=acc)[0] == (MMA if acc else TC)
    # one tile and one CTA of it for each KV head, joined by nobody else
    assert attention_form(16, 16, 64, F16, 9, 1, 8) == (MMA, 8, 1, True)
    # selected blocks: a problem for each token
    assert attention_form(32, 4, 128, F16, 50009, 8, 50001, blocks=30, block=32)[0] == MMA


def test_choose_forms():
    assert choose_form(506, 4) == CHOOSE[0] and choose_form(4086, 2) == CHOOSE[1] and choose_form(1557, 32) == CHOOSE[0]
    assert choose_form(8192, 19) == CHOOSE[0] and choose_form(8192, 18) == CHOOSE[1] and choose_form(8193, 19) == CHOOSE[2]
    assert choose_form(2**30, 65535) == CHOOSE[2] and choose_form(100, 65535) == CHOOSE[0]
