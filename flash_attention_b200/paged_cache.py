"""Bookkeeping of a paged KV cache and of trees of drafted tokens, on the GPU: nothing here synchronises, reads a length back or
allocates anything but its results, so that a step can be captured in a CUDA graph.

A step over a paged cache (block_table (batch, pages per sequence) int32, key j of sequence b in row j % page_block_size of page
block_table[b, j // page_block_size]; see flash_attn_with_kvcache) with drafted trees:

    slots, positions, cu_seqlens, seqlens = reserve_pages(block_table, lens, nodes, free_pages, num_free, page_block_size)
    words, positions = tree_layout(parents, lens)
    each layer:  q = rotary_axes_to_cache(q, k, v, cos, sin, positions, (pairs,), slots, k_cache, v_cache)
                 out = flash_attn_tree_with_kvcache(q, k_cache, v_cache, words, lens, block_table=block_table)
    the program picks the accepted path of each tree
    kept = keep_tree_path(all_caches, lens, path, nodes, block_table=block_table, seqlens=seqlens)
    release_pages(block_table, seqlens, kept, free_pages, num_free, page_block_size);  lens = kept

A sequence that had no room (seqlens == lens) has no slots, so that rotary_axes_to_cache stores nothing of it, and given seqlens, keep_tree_path keeps nothing
of it.  What attention says about it means nothing: the table's entries behind its last page are not its own.  Calls that store tokens by the table
(k and v of the attention calls) must not find them there: give those torch.where((seqlens > lens)[:, None], block_table, -1), where
-1 names no page, which is neither read nor written.

Not in this version of the reference, whose caches are one slab per sequence.
"""
from typing import Optional, Sequence, Union

import torch

import flash_attn_2_cuda as _ext

__all__ = ["reserve_pages", "release_pages", "tree_layout", "pack_tree_mask", "keep_tree_path"]


def reserve_pages(block_table, cache_seqlens, new_lens: Union[int, torch.Tensor], free_pages, num_free, page_block_size: int,
                  total: Optional[int] = None):
    """Room for new tokens: pages for them, and the slot and position of each.

    block_table: (batch, pages per sequence) int32, batch up to 16384; the new entries are written.
    cache_seqlens: (batch,) int32, tokens in the cache.  new_lens: (batch,) int32, tokens to come, or an int, as many for each.
    free_pages: (pool,) int32, a stack of unused pages; num_free: int32 [their number, 0], updated.  The second belongs to the
        call while it runs: calls that share a pool follow each other, on one stream or by events.
    total: rows of the packed new tokens, padding included; may be left out where new_lens is an int.

    Sequences are served in order; one gets its pages iff its table has room and they are there after all that the
    ones before it asked for (one that needs none always does).  Returns
    slots (total,) int64: page * page_block_size + row; -1 for the tokens of a sequence that had no room, and behind the last token;
    positions (total,) int32: of each token in its sequence, 0 behind the last token;
    cu_seqlens (batch + 1,) int32: sums of new_lens;
    seqlens (batch,) int32: lengths with the new tokens, or as they were where there was no room."""
    lens = new_lens if torch.is_tensor(new_lens) else None
    each = 0 if lens is not None else int(new_lens)
    if total is None:
        if lens is not None:
            raise RuntimeError("reserve_pages: total must be given where new_lens is a tensor")
        total = each * block_table.shape[0]
    return _ext._glue.reserve_pages(block_table, cache_seqlens, lens, each, free_pages, num_free, page_block_size, total)


def release_pages(block_table, cache_seqlens, keep_seqlens, free_pages, num_free, page_block_size: int):
    """The pages that cache_seqlens (batch,) tokens fill and the first keep_seqlens (batch,) of them do not go back on the stack
    (0: all of a sequence that has ended).  block_table is only read: its entries behind a sequence's last token mean nothing.
    Releasing what the last reserve_pages took leaves the stack as it was."""
    _ext._glue.release_pages(block_table, cache_seqlens, keep_seqlens, free_pages, num_free, page_block_size)


def tree_layout(parents, cache_seqlens):
    """parents: (batch, nodes) int32: of each node the node it hangs on, which must be an earlier one, or -1 for one that follows the
    tokens in the cache.  Any other value makes the node, and all that hangs on it, padding, which sees nothing of the tree and which nothing sees.
    Returns the words that flash_attn_tree_with_kvcache takes, (batch, nodes, ceil(nodes / 32)) int32: a node sees itself and the nodes it
    hangs on; and positions (batch, nodes) int32: cache_seqlens + the number of nodes above, -1 for padding."""
    return _ext._glue.tree_layout(parents, cache_seqlens)


def pack_tree_mask(mask):
    """The words of any mask: bool (batch or 1, nodes, nodes), [b, i, j]: node i sees node j."""
    return _ext._glue.pack_tree_mask(mask)


def keep_tree_path(caches: Union[Sequence[torch.Tensor], torch.Tensor], cache_seqlens, path, nodes: int, block_table: Optional[torch.Tensor] = None,
                   cache_batch_idx: Optional[torch.Tensor] = None, seqlens: Optional[torch.Tensor] = None):
    """After verification: the accepted nodes' rows move up behind the tokens in front of the tree, in all caches, in place.

    caches: K and V caches of any number of layers, of one shape, dtype and layout, paged with block_table, else a slab per sequence; or all of
        them as one tensor with the caches along its first dimension.
    path: (batch, longest) int32, the accepted nodes of each sequence from the top: each later than the one before and below `nodes`; any other
        value ends the path (pad with -1), and so does a node that is not in the caches, its row being past their capacity or in a page or slot
        that is not there.  Rows of the tree that are not on the path hold anything afterwards.
    seqlens: (batch,) int32, the lengths with the trees as reserve_pages gave them: a node whose row is not below ends the path.  Needed where a sequence may
        have had no room: what its table names behind its last page may be other sequences'.
    Returns cache_seqlens plus the number of accepted nodes, (batch,) int32.  Sequences must not share the rows that move."""
    return _ext._glue.keep_path(caches, cache_seqlens, path, nodes, block_table, cache_batch_idx, seqlens)
