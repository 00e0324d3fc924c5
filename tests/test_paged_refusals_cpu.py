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


def test_tangents_are_refused_not_lost():
    """A dual tensor of forward-mode differentiation does not require a gradient; the calls would give a result without a tangent."""
    import torch.autograd.forward_ad as fwd

    import flash_attention_b200 as fa
    from flash_attention_b200.layers.rotary import apply_rotary_emb_axes, rotary_axes_to_cache

    turn = dict(q=half(2, 7, 4, 64), k=half(2, 7, 2, 64), cos=half(30, 32), sin=half(30, 32), positions=i32(1, 2, 7), sections=(32,))
    store = dict(v=half(2, 7, 2, 64), slots=torch.zeros(14, dtype=torch.int64), k_cache=half(5, 16, 2, 64), v_cache=half(5, 16, 2, 64))
    tree = dict(q=half(2, 5, 4, 64), k_cache=half(2, 32, 2, 64), v_cache=half(2, 32, 2, 64), tree_mask=i32(2, 5, 1), cache_seqlens=i32(2))
    with fwd.dual_level():
        for name, call, args in [(n, apply_rotary_emb_axes, turn) for n in ("q", "k", "cos", "sin")] + [(n, rotary_axes_to_cache, {**turn, **store}) for n in "qkv"] + [
                (n, fa.flash_attn_tree_with_kvcache, tree) for n in ("q", "k_cache", "v_cache")]:
            for needs in (False, True):  # with a gradient as well
                dual = fwd.make_dual(args[name].clone().requires_grad_(needs), torch.ones_like(args[name]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(**{**args, name: dual})
        with pytest.raises(RuntimeError, match="CUDA"):  # nothing wrong but the device
            apply_rotary_emb_axes(**turn)


def test_in_place_to_cache_refuses_gradients():
    from flash_attention_b200.layers.rotary import rotary_axes_to_cache

    args = dict(k=half(2, 7, 2, 64), v=half(2, 7, 2, 64), cos=half(30, 32), sin=half(30, 32), positions=i32(1, 2, 7), sections=(32,),
                slots=torch.zeros(14, dtype=torch.int64), k_cache=half(5, 16, 2, 64), v_cache=half(5, 16, 2, 64))
    q = half(2, 7, 4, 64).requires_grad_(True)
    for x in (q, q * 1):
        with pytest.raises(RuntimeError, match="gradient"):
            rotary_axes_to_cache(x, inplace=True, **args)
    with pytest.raises(RuntimeError, match="CUDA"):  # nothing else is wrong without gradients, or out of place
        rotary_axes_to_cache(q, **args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        rotary_axes_to_cache(q, inplace=True, **args)


def test_one_column_may_have_any_stride():
    """A last dimension of one entry is contiguous whatever its stride says, which for a slice of a transposed tensor is not 1."""
    import flash_attention_b200 as fa

    args = dict(q=half(2, 5, 4, 64), k_cache=half(6, 64, 2, 64), v_cache=half(6, 64, 2, 64), cache_seqlens=i32(2))
    table, words = i32(3, 2).t()[:, :1], i32(1, 2, 5).permute(1, 2, 0)
    assert table.is_contiguous() and table.stride(1) != 1 and words.stride(2) != 1
    for kw in (dict(tree_mask=words), dict(tree_mask=i32(2, 5, 1), block_table=table), dict(tree_mask=words, block_table=table)):
        with pytest.raises(RuntimeError, match="CUDA"):  # nothing wrong but the device
            fa.flash_attn_tree_with_kvcache(**args, **kw)
    with pytest.raises(RuntimeError, match="words"):
        fa.flash_attn_tree_with_kvcache(**{**args, "q": half(2, 40, 4, 64)}, tree_mask=i32(2, 2, 40).transpose(1, 2))


def test_one_tensor_for_two_that_are_written():
    """Turned twice or not, K or V: which came last would decide."""
    import flash_attention_b200 as fa
    from flash_attention_b200.layers.rotary import apply_rotary_emb_axes, rotary_axes_to_cache

    x, c = half(2, 7, 2, 64), half(5, 16, 2, 64)
    turn = dict(cos=half(30, 32), sin=half(30, 32), positions=i32(1, 2, 7), sections=(32,))
    with pytest.raises(RuntimeError, match="twice"):
        apply_rotary_emb_axes(x, x, inplace=True, **turn)
    with pytest.raises(RuntimeError, match="CUDA"):  # out of place it is only read
        apply_rotary_emb_axes(x, x, **turn)
    store = dict(slots=torch.zeros(14, dtype=torch.int64), k_cache=c)
    with pytest.raises(RuntimeError, match="twice"):
        rotary_axes_to_cache(x, x, x, v_cache=c, **store, **turn)
    for k, v in ((x, x.clone()), (x.clone(), x)):  # read while q is written
        with pytest.raises(RuntimeError, match="twice"):
            rotary_axes_to_cache(x, k, v, v_cache=c.clone(), inplace=True, **store, **turn)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary_axes_to_cache(x, x, x, v_cache=c.clone(), **store, **turn)
    tree = dict(q=half(2, 5, 4, 64), tree_mask=i32(2, 5, 1), cache_seqlens=i32(2), k_cache=half(2, 32, 2, 64))
    new = dict(k=half(2, 5, 2, 64), v=half(2, 5, 2, 64))
    with pytest.raises(RuntimeError, match="twice"):
        fa.flash_attn_tree_with_kvcache(**tree, v_cache=tree["k_cache"], **new)
    with pytest.raises(RuntimeError, match="CUDA"):  # only read
        fa.flash_attn_tree_with_kvcache(**tree, v_cache=tree["k_cache"])


def test_c_entry_of_trees_refuses_rows_that_are_not_aligned(lib):
    """The kernels store new keys and values, and partial results, in 16-byte pieces."""
    import ctypes

    from flash_attention_b200 import _lib

    def tree(**kw):
        t = _lib.FaTreeArgs()
        a = t.kv
        a.batch = a.batch_cache = 2
        a.seqlen_q = a.seqlen_new = 5
        a.seqlen_cache, a.heads, a.heads_k, a.head_dim, a.dtype = 64, 4, 2, 64, 1
        a.window_left = a.window_right = -1
        a.cache_seqlens = a.softmax_lse = t.mask = 4096
        for name in ("q", "kcache", "vcache", "out", "knew", "vnew"):
            setattr(a, name, _lib.FaTensor(kw.get(name, 4096), kw.get(name + "_stride", 64 * 320), 128, 64))
        for name in ("num_splits", "lse_accum", "out_accum"):
            setattr(a, name, kw.get(name, 0))
        return lib.fa_fwd_tree(ctypes.byref(t), ctypes.c_void_p()), lib.fa_last_error()

    for kw, message in ((dict(knew=4098), b"knew: pointer"), (dict(vnew=4104), b"vnew: pointer"), (dict(knew_stride=1001), b"knew: strides"),
                        (dict(vnew=None), b"value"), (dict(num_splits=2, lse_accum=4096, out_accum=4100), b"out_accum: pointer")):
        rc, err = tree(**kw)
        assert rc == 1 and message in err, (kw, err)


def test_nothing_to_accept():
    from flash_attention_b200.generation import PagedInferenceParams

    params = PagedInferenceParams(1, 2, pages=8, pages_per_sequence=3, page_block_size=64, nheads_k=2, head_dim=64, dtype=torch.bfloat16, device="cpu")
    with pytest.raises(ValueError, match="accept: no step"):
        params.accept(i32(2, 3), 5)
