"""Block-table entries and slot numbers that name no page of the cache, one token per sequence: the token is dropped, the rows read as zeros, and
nothing outside the cache is read or written.  The caches are the middle of larger allocations, so that a stray address lands in pages that are looked at."""
import pytest
import torch

import flash_attention_b200 as fa
from flash_attention_b200 import _lib
from oracle import tree_oracle as TO

pytestmark = pytest.mark.gpu
GUARD, POOL, BATCH, PAGE = 6, 12, 4, 64


def guarded(rows, heads_k, dim, g):
    """A pool with GUARD pages in front of it and behind it, which hold values that would show in any result."""
    whole = torch.randn(GUARD + POOL + GUARD, rows, heads_k, dim, generator=g).bfloat16()
    whole[:GUARD], whole[GUARD + POOL:] = 1000.0, -1000.0
    return whole.cuda()


def check(out, lse, q, kc, vc, lens, **kw):
    """A token that sees itself and what is in front of it is a tree of one node."""
    sees = torch.ones(1, 1, 1, dtype=torch.bool)
    o, l, to, tl = TO.tree_attention(q.cpu(), kc.cpu(), vc.cpu(), sees, lens.cpu(), **kw)
    assert ((out.double().cpu() - o).abs() <= to).all()
    assert ((lse.double().cpu() - l).abs() <= tl).all()


# one token in the fused kernel (dims 64 and 128), behind kvcache_prep on the tensor cores (24 rows per KV head) and in the any-shape kernel
PATHS = [(8, 2, 128, "decode"), (4, 4, 64, "decode"), (48, 2, 128, "kvcache_prep+fwd_tc"), (8, 2, 96, "kvcache_prep+fwd_generic")]


@pytest.mark.parametrize("heads,heads_k,dim,path", PATHS)
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("paged", [True, False])
def test_one_token(heads, heads_k, dim, path, splits, paged):
    g = torch.Generator().manual_seed(dim + heads)
    rows = PAGE if paged else 3 * PAGE
    whole = [guarded(rows, heads_k, dim, g) for _ in range(2)]
    was = [w.clone() for w in whole]
    kc, vc = (w[GUARD:GUARD + POOL] for w in whole)
    lens = torch.tensor([70, 64, 130, 0], dtype=torch.int32)
    q = torch.randn(BATCH, 1, heads, dim, generator=g).bfloat16()
    k, v = (torch.randn(BATCH, 1, heads_k, dim, generator=g).bfloat16() for _ in range(2))
    if paged:
        table = torch.tensor([[3, -1, 5], [7, POOL, 0], [1, 2, POOL + GUARD - 1], [-GUARD, 4, 6]], dtype=torch.int32)
        place, kw = {}, dict(block_table=table)
    else:
        slots = torch.tensor([-1, 3, POOL, -GUARD], dtype=torch.int32)
        place, kw = {1: (3, 64)}, dict(cache_batch_idx=slots)
    out, lse = fa.flash_attn_with_kvcache(q.cuda(), kc, vc, k.cuda(), v.cuda(), cache_seqlens=lens.cuda(), causal=True, num_splits=splits, return_softmax_lse=True,
                                          **{n: t.cuda() for n, t in kw.items()})
    torch.cuda.synchronize()
    assert _lib.last_path().startswith(path), _lib.last_path()
    for w, x, new in zip(whole, was, (k, v)):
        for b, (slab, row) in place.items():
            x[GUARD + slab, row] = new[b, 0].cuda()
        assert torch.equal(w, x)
    check(out, lse, q, kc, vc, lens, **kw)


@pytest.mark.parametrize("heads,heads_k,dim,path", PATHS)
@pytest.mark.parametrize("splits", [1, 3])
def test_lengths_past_the_capacity(heads, heads_k, dim, path, splits):
    """Such a sequence sees the whole cache; its token is dropped."""
    g = torch.Generator().manual_seed(dim + heads)
    whole = [guarded(PAGE, heads_k, dim, g) for _ in range(2)]
    was = [w.clone() for w in whole]
    kc, vc = (w[GUARD:GUARD + POOL] for w in whole)
    table = torch.randperm(POOL, generator=g).view(BATCH, 3).int()
    lens = torch.tensor([192, 500, 10, 191], dtype=torch.int32)
    q = torch.randn(BATCH, 1, heads, dim, generator=g).bfloat16()
    k, v = (torch.randn(BATCH, 1, heads_k, dim, generator=g).bfloat16() for _ in range(2))
    out, lse = fa.flash_attn_with_kvcache(q.cuda(), kc, vc, k.cuda(), v.cuda(), cache_seqlens=lens.cuda(), causal=True, num_splits=splits, return_softmax_lse=True,
                                          block_table=table.cuda())
    assert _lib.last_path().startswith(path), _lib.last_path()
    for w, x, new in zip(whole, was, (k, v)):
        x[GUARD + int(table[2, 0]), 10], x[GUARD + int(table[3, 2]), 63] = new[2, 0].cuda(), new[3, 0].cuda()
        assert torch.equal(w, x)
    check(out, lse, q, kc, vc, lens, block_table=table)


@pytest.mark.parametrize("heads,heads_k,dim,path", [(4, 2, 128, "kvcache_prep+decode"), (16, 2, 64, "kvcache_prep+fwd_tc"), (4, 2, 40, "kvcache_prep+fwd_generic")])
@pytest.mark.parametrize("splits", [1, 3])
def test_several_tokens(heads, heads_k, dim, path, splits):
    """Five tokens, some of them in a page that is there and some not; a row of the table that names nothing, as for a sequence that had no room."""
    g = torch.Generator().manual_seed(dim)
    whole = [guarded(PAGE, heads_k, dim, g) for _ in range(2)]
    was = [w.clone() for w in whole]
    kc, vc = (w[GUARD:GUARD + POOL] for w in whole)
    lens = torch.tensor([62, 126, 100, 190], dtype=torch.int32)  # the last runs past the capacity
    table = torch.tensor([[3, -1, 5], [7, POOL, 0], [-1, -1, -1], [1, 2, 4]], dtype=torch.int32)
    q = torch.randn(BATCH, 5, heads, dim, generator=g).bfloat16()
    k, v = (torch.randn(BATCH, 5, heads_k, dim, generator=g).bfloat16() for _ in range(2))
    out, lse = fa.flash_attn_with_kvcache(q.cuda(), kc, vc, k.cuda(), v.cuda(), cache_seqlens=lens.cuda(), causal=False, num_splits=splits, return_softmax_lse=True,
                                          block_table=table.cuda())
    assert _lib.last_path().startswith(path), _lib.last_path()
    for w, x, new in zip(whole, was, (k, v)):
        for b in range(BATCH):
            for i in range(5):
                row = int(lens[b]) + i
                page = int(table[b, row // PAGE]) if row < 3 * PAGE else -1
                if 0 <= page < POOL:
                    x[GUARD + page, row % PAGE] = new[b, i].cuda()
        assert torch.equal(w, x)
    o, l, to, tl = TO.tree_attention(q, kc.cpu(), vc.cpu(), torch.ones(1, 5, 5, dtype=torch.bool), lens, block_table=table)
    assert ((out.double().cpu() - o).abs() <= to).all()
    assert ((lse.double().cpu() - l).abs() <= tl).all()
