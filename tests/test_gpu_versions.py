"""What the calls overwrite counts as changed for autograd: a backward pass that saved a value from before refuses to use it."""
import pytest
import torch

import flash_attention_b200 as fa
from flash_attention_b200 import paged_cache as pc
from flash_attention_b200.layers.rotary import apply_rotary_emb_axes, rotary_axes_to_cache

pytestmark = pytest.mark.gpu


def half(*shape):
    return torch.randn(shape, device="cuda").bfloat16()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def turn():
    return dict(q=half(1, 7, 4, 64), k=half(1, 7, 2, 64), cos=half(30, 32), sin=half(30, 32), positions=torch.arange(7, device="cuda")[None, None], sections=(32,))


def store():
    return dict(turn(), v=half(1, 7, 2, 64), slots=torch.arange(7, device="cuda"), k_cache=half(5, 16, 2, 64), v_cache=half(5, 16, 2, 64))


def tree(append=True):
    new = dict(k=half(2, 5, 2, 64), v=half(2, 5, 2, 64)) if append else {}
    return dict(q=half(2, 5, 4, 64), k_cache=half(2, 32, 2, 64), v_cache=half(2, 32, 2, 64), tree_mask=ints([[[31]] * 5] * 2), cache_seqlens=ints([3, 9]), **new)


def keep():
    return dict(caches=[half(2, 32, 2, 64), half(2, 32, 2, 64)], cache_seqlens=ints([3, 9]), path=ints([[1, 2]] * 2), nodes=4)


def pool():
    return dict(block_table=ints([[0, 1]] * 2), cache_seqlens=ints([3, 9]), free_pages=ints([4, 5, 6]), num_free=ints([3, 0]), page_block_size=64)


CALLS = [  # the call, its arguments, what it overwrites, what it leaves alone
    (lambda a: apply_rotary_emb_axes(**a, inplace=True), turn, ("q", "k"), ("cos", "positions")),
    (lambda a: apply_rotary_emb_axes(**a), turn, (), ("q", "k")),
    (lambda a: rotary_axes_to_cache(**a, inplace=True), store, ("q", "k_cache", "v_cache"), ("k", "v", "slots")),
    (lambda a: rotary_axes_to_cache(**a), store, ("k_cache", "v_cache"), ("q", "k", "v")),
    (lambda a: fa.flash_attn_tree_with_kvcache(**a), tree, ("k_cache", "v_cache"), ("q", "k", "v")),
    (lambda a: fa.flash_attn_tree_with_kvcache(**a), lambda: tree(False), (), ("q", "k_cache", "v_cache")),
    (lambda a: pc.keep_tree_path(**a), keep, ("caches",), ("path", "cache_seqlens")),
    (lambda a: pc.keep_tree_path(**a), lambda: dict(keep(), caches=half(3, 2, 32, 2, 64)), ("caches",), ("path",)),
    (lambda a: pc.reserve_pages(**a, new_lens=70), pool, ("block_table", "num_free"), ("cache_seqlens",)),
    (lambda a: pc.release_pages(**a, keep_seqlens=ints([0, 0])), pool, ("free_pages", "num_free"), ("block_table",)),
]


@pytest.mark.parametrize("which", range(len(CALLS)))
def test_versions(which):
    call, make, written, read = CALLS[which]
    args = make()
    flat = lambda names: [t for n in names for t in (args[n] if isinstance(args[n], list) else [args[n]])]  # noqa: E731
    before = [t._version for t in flat(written + read)]
    call(args)
    after = [t._version for t in flat(written + read)]
    n = len(flat(written))
    assert all(b > a for a, b in zip(before[:n], after[:n])) and before[n:] == after[n:]


def test_a_saved_value_that_is_turned_in_place_is_noticed():
    w = half(64).requires_grad_(True)
    for name in ("q", "k"):
        args = turn()
        y = (args[name] * w).sum()
        apply_rotary_emb_axes(**args, inplace=True)
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward()
    args = store()
    y = (args["q"] * w).sum() + (args["k_cache"][2] * w).sum()
    rotary_axes_to_cache(**args)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()


def test_inference_tensors_are_taken_as_before():
    for make, call, _, _ in ((m, c, w, r) for c, m, w, r in CALLS):
        with torch.inference_mode():
            args = make()
            call(args)
        with torch.no_grad():
            call(args)
