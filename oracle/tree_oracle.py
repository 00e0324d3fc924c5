"""Drafted trees over a (paged) KV cache, positions with several axes and the bookkeeping of pages, restated plainly on the CPU in 64 bits
(whole numbers: in python), with bounds on how far a kernel that keeps its sums in 32 bits may be off."""
import math

import torch


def half_step(dtype):
    """The largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def cache_rows(cache, b, n, block_table=None, cache_batch_idx=None):
    """Rows [0, n) of sequence b of a cache, (n, heads_k, dim); pages or slots that are not there read as zeros."""
    if block_table is None:
        slot = b if cache_batch_idx is None else int(cache_batch_idx[b])
        return cache[slot, :n] if 0 <= slot < cache.shape[0] else torch.zeros_like(cache[0, :n])
    ps = cache.shape[1]
    pages = block_table[b, : -(-n // ps)].tolist()
    parts = [cache[p] if 0 <= p < cache.shape[0] else torch.zeros_like(cache[0]) for p in pages]
    return torch.cat(parts)[:n] if parts else cache[0, :0]


def tree_attention(q, k_cache, v_cache, sees, lens, block_table=None, cache_batch_idx=None, scale=None):
    """q (batch, nodes, heads, dim); sees (batch or 1, nodes, nodes) bool.  Returns out and lse in 64 bits, and for each how far a kernel may be off.

    The kernels keep scores, maximum and sum in 32 bits and round the weights p of a row to the type of V before they multiply them.  With u half a
    step of that type: a weight is off by u of itself (fp16: by 2^-25 of the largest where it is subnormal), a score by (dim + 8) 2^-24 sum |q k|
    (every addition and the scale), an exponential by 2^-20, the sum of n weights by n 2^-24; the result is rounded once more."""
    batch, nodes, heads, dim = q.shape
    heads_k = k_cache.shape[2]
    group = heads // heads_k
    cap = block_table.shape[1] * k_cache.shape[1] if block_table is not None else k_cache.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, lse = torch.zeros(batch, nodes, heads, dim, dtype=torch.float64), torch.full((batch, heads, nodes), math.inf, dtype=torch.float64)
    tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    u = half_step(q.dtype)
    for b in range(batch):
        base = min(max(int(lens[b]), 0), cap)
        n = min(base + nodes, cap)
        k = cache_rows(k_cache, b, n, block_table, cache_batch_idx).double()
        v = cache_rows(v_cache, b, n, block_table, cache_batch_idx).double()
        on = torch.ones(nodes, n, dtype=torch.bool)
        m = sees[b % sees.shape[0]]
        on[:, base:] = m[:, : n - base]
        used = on.any(0)
        k, v = torch.where(used[:, None, None], k, 0.0), torch.where(used[:, None, None], v, 0.0)  # (what nobody sees may be NaN)
        qs = q[b].double().view(nodes, heads_k, group, dim)
        s = torch.einsum("thgd,khd->thgk", qs, k) * scale
        mag = torch.einsum("thgd,khd->thgk", qs.abs(), k.abs()) * scale
        s = torch.where(on[:, None, None], s, -math.inf)
        top = s.amax(-1, keepdim=True)
        some = top > -math.inf
        p = torch.where(on[:, None, None], torch.exp(s - torch.where(some, top, 0.0)), 0.0)
        total = p.sum(-1, keepdim=True)
        w = p / torch.where(some, total, 1.0)
        o = torch.einsum("thgk,khd->thgd", w, v)
        a = torch.einsum("thgk,khd->thgd", w, v.abs())
        ds = (torch.where(on[:, None, None], mag, 0.0).amax(-1, keepdim=True) * (dim + 8) * 2.0 ** -24)
        e32 = ds + n * 2.0 ** -24 + 2.0 ** -20
        t = u * (a + o.abs()) + 2 * e32 * a
        if q.dtype == torch.float16:
            t = t + 2.0 ** -25 * torch.einsum("thgk,khd->thgd", on[:, None, None].double().expand_as(w), v.abs()) + 2.0 ** -25
        out[b], tol_o[b] = o.reshape(nodes, heads, dim), t.reshape(nodes, heads, dim)
        row = torch.where(some, top + torch.log(torch.where(some, total, 1.0)), math.inf)[..., 0]
        lse[b] = row.reshape(nodes, heads).T
        tol_l[b] = (e32[..., 0] + 2.0 ** -20 * torch.where(some[..., 0], row.abs(), 0.0)).reshape(nodes, heads).T
    return out, lse, tol_o, tol_l


def axis_of_pairs(sections, cycled):
    axes, pairs = len(sections), sum(sections)
    if not cycled:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    of = [0] * pairs
    for a in range(1, axes):
        for j in range(sections[a]):
            of[a + axes * j] = a
    return of


def turn(x, cos, sin, positions, sections, cycled=False, interleaved=False, conjugate=False):
    """x (..., heads, dim), positions (axes, ...).  Returns the turned rows in 64 bits and how far a kernel may be off that computes in 32 bits (two
    products and a sum: 2^-23 of their magnitudes) and rounds once."""
    pairs = cos.shape[1]
    out, mag = x.double().clone(), x.double().abs()
    for i, a in enumerate(axis_of_pairs(sections, cycled)):
        at = positions[a].long()
        inside = (at >= 0) & (at < cos.shape[0])
        row = at.clamp(0, max(cos.shape[0] - 1, 0))
        c = torch.where(inside, cos[row, i].double(), 1.0)[..., None] if cos.shape[0] else torch.ones_like(at, dtype=torch.float64)[..., None]
        s = torch.where(inside, sin[row, i].double(), 0.0)[..., None] if cos.shape[0] else torch.zeros_like(at, dtype=torch.float64)[..., None]
        s = -s if conjugate else s
        i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        a0, a1 = x[..., i0].double(), x[..., i1].double()
        out[..., i0], out[..., i1] = a0 * c - a1 * s, a0 * s + a1 * c
        mag[..., i0], mag[..., i1] = (a0 * c).abs() + (a1 * s).abs(), (a0 * s).abs() + (a1 * c).abs()
    tol = half_step(x.dtype) * out.abs() + 2.0 ** -22 * mag
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    return out, tol


class Pool:
    """Unused pages, and the tables they go to."""

    def __init__(self, free, num_free, page):
        self.free, self.n, self.page = list(free), num_free, page

    def pages(self, tokens):
        return -(-tokens // self.page)

    def reserve(self, table, lens, new, total):
        asked, slots, positions, cu, seqlens = 0, [-1] * total, [0] * total, [0], []
        pages_left, taken_total = self.n, 0
        t = 0
        for b, (length, n) in enumerate(zip(lens, new)):
            have, want = self.pages(length), self.pages(length + n)
            need = want - have if want <= len(table[b]) else 0
            room = want <= len(table[b]) and (need == 0 or asked + need <= pages_left)
            if room:
                for i in range(need):
                    table[b][have + i] = self.free[pages_left - 1 - asked - i]
                taken_total = max(taken_total, asked + need) if need else taken_total
            asked += need
            for i in range(n):
                if t < total:
                    pos = length + i
                    positions[t] = pos
                    slots[t] = table[b][pos // self.page] * self.page + pos % self.page if room else -1
                t += 1
            cu.append(t)
            seqlens.append(length + n if room else length)
        self.n = pages_left - taken_total
        return slots, positions, cu, seqlens

    def release(self, table, lens, keep):
        back = []
        for b, (length, k) in enumerate(zip(lens, keep)):
            back += table[b][self.pages(min(k, length)):self.pages(length)]
        for i, page in enumerate(back):
            self.free[self.n + len(back) - 1 - i] = page
        self.n += len(back)


def ancestors(parents):
    """parents: list of lists.  (batch, nodes, nodes) bool and the number of nodes above, -1 for nodes that are not there."""
    nodes = len(parents[0])
    sees, above = torch.zeros(len(parents), nodes, nodes, dtype=torch.bool), torch.full((len(parents), nodes), -1)
    for b, row in enumerate(parents):
        for i in range(nodes):
            chain, j = [i], i
            while 0 <= row[j] < j:
                j = row[j]
                chain.append(j)
            if row[j] == -1:
                sees[b, i, chain] = True
                above[b, i] = len(chain) - 1
    return sees, above


def pack_words(sees):
    nodes = sees.shape[-1]
    w = torch.zeros(*sees.shape[:-1], (nodes + 31) // 32, dtype=torch.int64)
    for j in range(nodes):
        w[..., j // 32] |= sees[..., j].long() << (j % 32)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def keep(cache_of, lens, path, nodes, cap):
    """cache_of(b, row) -> key of a place, None for one that is not there; returns the moves [(from, to)] of every sequence in order, and the new lengths.  A
    path ends at the first node that does not go on, or whose row, or the row it moves to, is not there."""
    there = lambda b, row: 0 <= row < cap and cache_of(b, row) is not None  # noqa: E731
    moves, new = [], []
    for b, (length, steps) in enumerate(zip(lens, path)):
        last, n = -1, 0
        for node in steps:
            if not (last < node < nodes) or not there(b, length + node) or not there(b, length + n):
                break
            if node != n:
                moves.append((cache_of(b, length + node), cache_of(b, length + n)))
            last, n = node, n + 1
        new.append(length + n)
    return moves, new
