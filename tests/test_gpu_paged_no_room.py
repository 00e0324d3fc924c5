"""PagedSelfAttention for sequences that got no room: zeros, whatever their tables name, and the other sequences as if they were alone.  Pages go back once."""
import pytest
import torch

from flash_attention_b200.generation import PagedInferenceParams, PagedSelfAttention

pytestmark = pytest.mark.gpu


# rows per KV head for the few-row kernel, the tensor-core kernel and the any-shape kernel
@pytest.mark.parametrize("heads,heads_k,dim", [(4, 2, 64), (32, 2, 128), (2, 1, 40)])
@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("nodes", [1, 6, 40])
def test_zeros(heads, heads_k, dim, tree, nodes):
    make = lambda batch, pages: PagedInferenceParams(1, batch, pages, 4, 64, heads_k, dim, torch.bfloat16, "cuda")  # noqa: E731
    params, alone = make(3, 4), make(1, 2)
    for p in (params, alone):
        p.caches.fill_(float("nan"))
    layer = PagedSelfAttention(0, dim, (dim // 2,), 300, device="cuda")
    g = torch.Generator().manual_seed(nodes)
    x = lambda n: [torch.randn(3, n, h, dim, generator=g).bfloat16().cuda() for h in (heads, heads_k, heads_k)]  # noqa: E731
    parents = torch.arange(-1, nodes - 1, dtype=torch.int32, device="cuda").expand(3, -1)

    first = x(64)  # a page each; one is left
    for p, rows in ((params, first), (alone, [t[:1] for t in first])):
        p.begin(64)
        layer(*rows, p)
    params.block_table[1:, 1] = params.block_table[0, 0]  # what an earlier use of the table left there: a page of another sequence
    assert params.num_free.tolist() == [1, 0]
    rows, before = x(nodes), params.caches.clone()
    for p in (params, alone):
        p.begin_tree(parents[: p.lengths.shape[0]]) if tree else p.begin(nodes)
    assert params.seqlens.tolist() == [64 + nodes, 64, 64]
    out, want = layer(*rows, params), layer(*[t[:1] for t in rows], alone)
    assert not out[1:].any() and want.any() and not torch.isnan(want).any()
    # (The keys may be cut into other parts.  Each side rounds the weights, whose sum is 1, and the result: two half steps of the largest value.)
    largest = max(first[2].float().abs().max(), rows[2].float().abs().max())
    assert (out[:1].float() - want.float()).abs().max() <= 2.1 * torch.finfo(torch.bfloat16).eps * largest
    own = params.block_table[0, 1].item()
    now = params.caches.clone()
    now[:, :, own], before[:, :, own] = 0, 0
    assert torch.equal(now.nan_to_num(7.0), before.nan_to_num(7.0))
    if tree:
        params.accept(torch.zeros(3, 1, dtype=torch.int32, device="cuda"), nodes)
        assert params.lengths.tolist() == [65, 64, 64]
    # two pages come free: the second sequence gets its turn, the third does not
    params.end(torch.tensor([True, False, False], device="cuda"))
    params.begin(1)
    assert params.seqlens.tolist() == [1, 65, 64]
    out = layer(*x(1), params)
    assert out[:2].any(-1).all() and not torch.isnan(out).any() and not out[2].any()


def test_a_table_that_is_full():
    """A sequence that outgrows its table, beside one that does not."""
    params = PagedInferenceParams(1, 2, 10, 2, 64, 2, 64, torch.bfloat16, "cuda")
    layer = PagedSelfAttention(0, 64, (32,), 128, device="cuda")
    g = torch.Generator().manual_seed(0)
    x = lambda n: [torch.randn(2, n, h, 64, generator=g).bfloat16().cuda() for h in (4, 2, 2)]  # noqa: E731
    params.begin(100)
    layer(*x(100), params)
    params.end(torch.tensor([False, True], device="cuda"))
    params.begin_tree(torch.arange(-1, 29, dtype=torch.int32, device="cuda").expand(2, -1))
    out = layer(*x(30), params)
    assert params.seqlens.tolist() == [100, 30] and not out[0].any() and out[1].any(-1).all()
    params.accept(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), 30)
    assert params.lengths.tolist() == [100, 1]


def test_a_step_is_accepted_once():
    """A second accept, or one behind end(), would put the same pages on the stack again."""
    params = PagedInferenceParams(1, 2, 10, 4, 64, 2, 64, torch.bfloat16, "cuda")
    path = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    parents = torch.arange(-1, 69, dtype=torch.int32, device="cuda").expand(2, -1)
    for after in (lambda: params.accept(path, 70), lambda: params.end(torch.tensor([True, False], device="cuda"))):
        params.begin_tree(parents)
        assert params.num_free[0] < 8
        after()
        lengths, num = params.lengths.tolist(), params.num_free.tolist()
        with pytest.raises(ValueError, match="accept"):
            params.accept(path, 70)
        assert params.lengths.tolist() == lengths and params.num_free.tolist() == num
    stack = params.free_pages[: params.num_free[0]].tolist()
    assert len(set(stack)) == len(stack)
    # a chain of drafts after begin() is accepted like a tree
    params.begin(3)
    params.accept(torch.tensor([[0, 1], [0, -1]], dtype=torch.int32, device="cuda"), 3)
    assert params.lengths.tolist() == [lengths[0] + 2, lengths[1] + 1]
