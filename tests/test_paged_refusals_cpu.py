"""What the calls on paged caches, trees and positions with several axes refuse, beside test_trees_cpu.py."""
import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def lib():
    from flash_attention_b200 import _lib
    from flash_attention_b200.csrc import build as b

    b.build()
    return _lib.lib()


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def half(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("seqlens,message", [(i32(3), "seqlens"), (i32(2).long(), "seqlens"), (i32(4)[::2], "seqlens"), (i32(2), "CUDA")])
def test_keep_refuses_lengths(seqlens, message):
    from flash_attention_b200 import paged_cache as pc

    with pytest.raises(RuntimeError, match=message):
        pc.keep_tree_path([half(2, 64, 2, 64)], i32(2), i32(2, 3), 4, seqlens=seqlens)
