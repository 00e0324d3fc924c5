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


def test_rotary_tables_shorter_than_a_sequences_pages():
    """Tokens outside the tables are not turned: where the layer makes the positions itself it has to have a row for each."""
    from flash_attention_b200.generation import PagedInferenceParams, PagedSelfAttention

    params = PagedInferenceParams(1, 2, pages=8, pages_per_sequence=3, page_block_size=64, nheads_k=2, head_dim=64, dtype=torch.bfloat16, device="cpu")
    params.slots, params.positions = torch.zeros(10, dtype=torch.int64), i32(2, 5)
    call = lambda rows, **kw: PagedSelfAttention(0, 64, (32,), rows)(half(2, 5, 4, 64), half(2, 5, 2, 64), half(2, 5, 2, 64), params, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="max_position 191 is less than the 192"):
        call(191)
    with pytest.raises(RuntimeError, match="CUDA"):  # nothing wrong but the device
        call(192)
    with pytest.raises(RuntimeError, match="CUDA"):  # positions of the caller's own
        call(191, positions=i32(1, 2, 5))
