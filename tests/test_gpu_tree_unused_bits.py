"""Bits of a tree's words behind its last node say nothing: rows of the cache behind the tree, which hold NaN or large values here, stay unseen."""
import pytest
import torch

import flash_attention_b200 as fa
from flash_attention_b200 import _lib
from oracle import tree_oracle as TO

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [float("nan"), 1000.0])
@pytest.mark.parametrize("path,nodes,heads,heads_k,dim", [("decode", 5, 4, 2, 64), ("decode", 3, 6, 3, 16), ("decode", 16, 1, 1, 256), ("fwd_tc", 40, 4, 2, 128),
                                                          ("fwd_tc", 37, 2, 2, 8), ("fwd_tc", 64, 2, 2, 192), ("fwd_tc", 65, 8, 2, 64), ("fwd_generic", 5, 4, 2, 64),
                                                          ("fwd_generic", 40, 4, 2, 128)])
@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("splits", [1, 3])
def test_rows_behind_the_tree(path, nodes, heads, heads_k, dim, page, splits, value, monkeypatch):
    if path == "fwd_generic":
        monkeypatch.setenv("FA_B200_FORCE_GENERIC", "1")
    g = torch.Generator().manual_seed(nodes)
    lens = torch.tensor([0, 100, 61, 64], dtype=torch.int32)
    cap = 320
    sees = torch.rand(4, nodes, nodes, generator=g) < 0.4
    q = torch.randn(4, nodes, heads, dim, generator=g).half()
    caches = [torch.randn(4, cap, heads_k, dim, generator=g).half() for _ in range(2)]
    for c in caches:
        for b in range(4):
            c[b, int(lens[b]) + nodes:] = value
    ref = TO.tree_attention(q, *caches, sees, lens)
    table = None
    if page:
        table = torch.randperm(4 * cap // page, generator=g).view(4, -1).int()
        pools = [torch.empty_like(c).view(-1, page, heads_k, dim) for c in caches]
        for pool, c in zip(pools, caches):
            pool[table.long().flatten()] = c.view(-1, page, heads_k, dim)
        caches = pools
    words = TO.pack_words(sees)
    if nodes % 32:
        words[..., -1] |= -1 << (nodes % 32)
    out, lse = fa.flash_attn_tree_with_kvcache(q.cuda(), caches[0].cuda(), caches[1].cuda(), words.cuda(), lens.cuda(), block_table=None if table is None else table.cuda(),
                                               num_splits=splits, return_softmax_lse=True)
    assert _lib.last_path().startswith(path), _lib.last_path()
    out, lse = out.double().cpu(), lse.double().cpu()
    o, l, to, tl = ref
    assert ((out - o).abs() <= to).all()
    assert torch.equal(lse.isinf(), l.isinf()) and ((lse - l).abs()[~l.isinf()] <= tl[~l.isinf()]).all()
