"""keep_tree_path where the accepted nodes, or the rows they move to, are not in the caches or not the sequence's: the path ends there, in the caches and
in the lengths."""
import pytest
import torch

from flash_attention_b200 import paged_cache as pc

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cache(*shape):
    return torch.randint(-1000, 1000, shape, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("paged", [True, False])
def test_a_node_past_the_capacity_ends_the_path(paged):
    """192 rows, 185 of them taken: nodes 0 to 6 were stored, node 10 was not."""
    table = ints([[2, 0, 1]]) if paged else None
    c = cache(3, 64, 2, 64) if paged else cache(1, 192, 2, 64)
    rows = lambda: torch.cat([c[p] for p in (2, 0, 1)]) if paged else c[0]  # noqa: E731
    was = rows().clone()
    for path, kept, moves in (([0, 10], 186, {}), ([10], 185, {}), ([2, 6, 7], 187, {185: 187, 186: 191}), ([0, 1, 2, 3, 4, 5, 6, 7], 192, {})):
        for t, x in zip((c[2], c[0], c[1]) if paged else (c[0][:64], c[0][64:128], c[0][128:]), was.split(64)):
            t.copy_(x)
        assert pc.keep_tree_path([c], ints([185]), ints([path]), 12, block_table=table).tolist() == [kept]
        want = was.clone()
        for to, at in moves.items():
            want[to] = was[at]
        assert torch.equal(rows(), want)


def test_lengths_at_and_past_the_capacity_and_below_zero():
    c = cache(4, 64, 2, 64)
    was = c.clone()
    assert pc.keep_tree_path([c], ints([64, 100, -3, 2 ** 31 - 2]), ints([[0, 1]] * 4), 3).tolist() == [64, 100, -3, 2 ** 31 - 2]
    assert torch.equal(c, was)


def test_pages_and_slots_that_are_not_there():
    """The page of a node, or of the row it would move to."""
    c = cache(6, 64, 2, 64)
    was = c.clone()
    table = ints([[3, -1, 4], [-1, 5, 0], [0, 6, 1], [1, 2, 3]])
    lens, path = ints([60, 62, 62, 62]), ints([[0, 3, 5], [1, 2, 3], [0, 1, 2], [0, 2, 3]])
    # 0: rows 60, 63, then a row of the missing page; 1: its first target is missing; 2: rows 62, 63, then a missing one; 3: all there
    assert pc.keep_tree_path([c], lens, path, 8, block_table=table).tolist() == [62, 62, 64, 65]
    want = was.clone()
    want[3, 61] = was[3, 63]
    want[1, 63], want[2, 0] = was[2, 0], was[2, 1]
    assert torch.equal(c, want)
    c.copy_(was)
    assert pc.keep_tree_path([c], ints([10, 10, 10]), ints([[1, 2]] * 3), 8, cache_batch_idx=ints([5, -1, 6])).tolist() == [12, 10, 10]
    want = was.clone()
    want[5, 10], want[5, 11] = was[5, 11], was[5, 12]
    assert torch.equal(c, want)


@pytest.mark.parametrize("depth", [31, 32, 33, 64, 65, 100])
def test_long_paths_that_end_at_the_capacity(depth):
    """The end in the first, the second and the third group of 32 nodes, and at their borders."""
    nodes = 2 * depth
    for room in (1, depth, 2 * depth - 1, 2 * depth):
        c = cache(1, 20 + room, 1, 8)
        was = c.clone()
        path = list(range(1, nodes, 2))
        kept = sum(node < room for node in path)
        assert pc.keep_tree_path([c], ints([20]), ints([path]), nodes).tolist() == [20 + kept]
        want = was.clone()
        want[0, 20:20 + kept] = was[0, 21:21 + 2 * kept:2]
        assert torch.equal(c, want)


def test_a_sequence_that_had_no_room_leaves_the_others_pages_alone():
    """The second sequence gets no page; what its table names behind its own page belongs to the first one and to nobody."""
    c = cache(5, 64, 2, 64)
    table, lens = ints([[3, 1], [2, 3]]), ints([60, 61])
    free, num = ints([4, 0]), ints([1, 0])  # the stack's first entry: one page for two that want one
    slots, _, _, seqlens = pc.reserve_pages(table, lens, 8, free, num, 64)
    assert seqlens.tolist() == [68, 61] and table.tolist() == [[3, 4], [2, 3]] and slots[8:].tolist() == [-1] * 8
    was = c.clone()
    path = ints([[1, 4, 5], [1, 4, 5]])
    kept = pc.keep_tree_path([c], lens, path, 8, block_table=table, seqlens=seqlens)
    want = was.clone()
    want[3, 60], want[3, 61], want[3, 62] = was[3, 61], was[4, 0], was[4, 1]
    assert kept.tolist() == [63, 61] and torch.equal(c, want)
    # lengths in the middle of a path, and without caches
    assert pc.keep_tree_path([], lens, path, 8, seqlens=ints([65, 62])).tolist() == [62, 61]
    # tokens stored by the call: not with a table that names no page for it
    import flash_attention_b200 as fa

    q, k = torch.randn(2, 8, 4, 64, device="cuda").bfloat16(), torch.randn(2, 8, 2, 64, device="cuda").bfloat16()
    words = pc.pack_tree_mask(torch.ones(1, 8, 8, dtype=torch.bool, device="cuda"))
    kc, vc = c.clone(), c.clone()
    mine = torch.where((seqlens > lens)[:, None], table, -1)
    fa.flash_attn_tree_with_kvcache(q, kc, vc, words, lens, k=k, v=k, block_table=mine)
    want = c.clone()
    want[3, 60:64], want[4, :4] = k[0, :4], k[0, 4:]
    assert torch.equal(kc, want) and torch.equal(vc, want)


@pytest.mark.parametrize("dim", [8, 6])  # in pieces of 16 bytes, and of two
@pytest.mark.parametrize("depth", [2560, 2561, 3071, 3073, 12288])
def test_the_longest_paths(depth, dim):
    """Around the shared memory that a launch has without asking, and the most there may be."""
    c = cache(1, 2 * depth + 5, 1, dim)
    was = c.clone()
    path = torch.arange(1, 2 * depth, 2, device="cuda").int()[None]
    assert pc.keep_tree_path([c], ints([3]), path, 2 * depth).tolist() == [3 + depth]
    want = was.clone()
    want[0, 3:3 + depth] = was[0, 4:4 + 2 * depth:2]
    assert torch.equal(c, want)
    with pytest.raises(RuntimeError, match="12288"):
        pc.keep_tree_path([c], ints([3]), torch.zeros(1, 12289, dtype=torch.int32, device="cuda"), 2 * depth)
