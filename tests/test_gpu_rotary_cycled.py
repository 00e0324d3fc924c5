"""Axes that take turns (cycled): q and k, forward, both gradients and on the way into a cache, against the definition in 64 bits and, since the order of
the pairs is all that is different, against sections in a row."""
import pytest
import torch

from flash_attention_b200.layers.rotary import apply_rotary_emb_axes, rotary_axes_to_cache
from oracle import tree_oracle as TO

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
CASES = [  # lead, heads, heads_k, dim, sections
    ((2, 21), 4, 2, 128, (24, 20, 20)),
    ((70,), 6, 3, 128, (44, 10, 10)),
    ((2, 9), 3, 1, 80, (16, 12, 12)),
    ((33,), 5, 5, 72, (10, 9, 9, 8)),
    ((33,), 2, 1, 96, (7, 6)),
    ((1, 1), 32, 8, 64, (11, 11, 10)),
    ((40,), 4, 2, 50, (3, 2)),
]


def make(lead, heads, heads_k, dim, sections, dtype, count):
    g = torch.Generator().manual_seed(dim + len(lead))
    angle = torch.rand(53, sum(sections), generator=g) * 6.3
    pos = torch.randint(-2, 56, (len(sections),) + lead, generator=g).int()  # some outside the tables
    rows = [torch.randn(lead + (h, dim), generator=g).to(DT[dtype]) for h in (heads, heads_k, heads, heads_k)[:count]]
    return angle.cos().to(DT[dtype]), angle.sin().to(DT[dtype]), pos, rows, g


def close(x, want, what):
    out, tol = want
    assert ((x.detach().double().cpu() - out).abs() <= tol).all(), what


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,heads,heads_k,dim,sections", CASES)
def test_forward_and_backward(lead, heads, heads_k, dim, sections, interleaved, dtype):
    cos, sin, pos, (q, k, dq, dk), _ = make(lead, heads, heads_k, dim, sections, dtype, 4)
    how = dict(cycled=True, interleaved=interleaved)
    qd, kd = q.cuda().requires_grad_(True), k.cuda().requires_grad_(True)
    qr, kr = apply_rotary_emb_axes(qd, kd, cos.cuda(), sin.cuda(), pos.cuda(), sections, **how)
    gq, gk = torch.autograd.grad((qr, kr), (qd, kd), (dq.cuda(), dk.cuda()))
    for x, of, back in ((qr, q, False), (kr, k, False), (gq, dq, True), (gk, dk, True)):
        close(x, TO.turn(of, cos, sin, pos, sections, conjugate=back, **how), back)
    # the same angles from sections in a row, the pairs sorted by their axes
    of = torch.tensor(TO.axis_of_pairs(sections, True))
    if not interleaved:
        order = torch.argsort(of, stable=True)
        pairs = sum(sections)
        cols = torch.cat([order, order + pairs, torch.arange(2 * pairs, dim)])
        got, _ = apply_rotary_emb_axes(q[..., cols].contiguous().cuda(), None, cos[:, order].contiguous().cuda(), sin[:, order].contiguous().cuda(), pos.cuda(),
                                       [int((of == a).sum()) for a in range(len(sections))])
        assert torch.equal(got, qr.detach()[..., cols.cuda()])


def test_gradient_against_differences():
    """Linear: f(x + e) - f(x - e) = 2 turn(e); whole numbers and quarter turns, which 16 bits hold."""
    sections = (3, 3, 2)
    turns = torch.arange(6)[:, None] + torch.arange(8)
    cos, sin = torch.tensor([1.0, 0.0, -1.0, 0.0])[turns % 4].half().cuda(), torch.tensor([0.0, 1.0, 0.0, -1.0])[turns % 4].half().cuda()
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 6, (3, 5), generator=g).cuda()
    x, w = (torch.randint(-8, 9, (5, 2, 16), generator=g).half().cuda() for _ in range(2))
    f = lambda t: apply_rotary_emb_axes(t, None, cos, sin, pos, sections, cycled=True)[0]  # noqa: E731
    leaf = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(f(leaf), leaf, w)
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), dtype=x.dtype, device="cuda")
        e[i] = 1
        e = e.view_as(x)
        assert ((f(x + e) - f(x - e)) * w).double().sum() / 2 == gx.flatten()[i].double()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,heads,heads_k,dim,sections", CASES)
def test_to_cache(lead, heads, heads_k, dim, sections, interleaved, dtype):
    cos, sin, pos, (q, k, _, v), g = make(lead, heads, heads_k, dim, sections, dtype, 4)
    how = dict(cycled=True, interleaved=interleaved)
    n = k[..., 0, 0].numel()
    pages = -(-n // 16) + 2
    kc, vc = (torch.randn(pages, 16, heads_k, dim, generator=g).to(DT[dtype]) for _ in range(2))
    slots = torch.randperm(pages * 16, generator=g)[:n]
    slots[1::7] = -1
    kd, vd = kc.cuda(), vc.cuda()
    r = rotary_axes_to_cache(q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), pos.cuda(), sections, slots.cuda(), kd, vd, **how)
    close(r, TO.turn(q, cos, sin, pos, sections, **how), "q")
    out, tol = TO.turn(k, cos, sin, pos, sections, **how)
    real = slots >= 0
    want, slack = kc.double().view(-1, heads_k, dim), torch.zeros(pages * 16, heads_k, dim, dtype=torch.float64)
    want[slots[real]], slack[slots[real]] = out.reshape(n, heads_k, dim)[real], tol.reshape(n, heads_k, dim)[real]
    assert ((kd.double().cpu().view(-1, heads_k, dim) - want).abs() <= slack).all()
    vc.view(-1, heads_k, dim)[slots[real]] = v.reshape(n, heads_k, dim)[real]
    assert torch.equal(vd.cpu(), vc)
