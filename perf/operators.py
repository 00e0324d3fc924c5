"""The calls that verify drafted token trees over a (paged) KV cache, and the positions with several axes that go with
them, as data: sizes, inputs, one pass each, the operators' plain forms and their definition in 64 bits.

Sizes are those of this repository's benchmark and tests and between them: 32/8 heads of 128 for serving, caches of up to
16384 tokens here, pages of 64 to 256 rows, odd ones beside them.
"""
import math
import random

import torch

own = False  # whether run() makes the framework's calls or computes the plain form

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


# ----------------------------------------------------------------------------------------------- cases
def _tree(name, **kw):
    """Attention of `nodes` drafted tokens per sequence, of which each sees the cache and its ancestors.  page: rows of a
    page, 0 for one slab per sequence.  append: the drafted tokens' k and v are put into the cache by the same call."""
    c = dict(op="tree", batch=1, nodes=8, heads=32, heads_k=8, dim=128, dtype="bf16", len_lo=0, len_hi=1024, page=0, append=False)
    return _named(name, c, kw)


def _rope(name, **kw):
    """Rotary positions with several axes on q and k, forward and backward.  batch 0: packed tokens.  sections: pairs of
    each axis.  span: rows of the tables."""
    c = dict(op="rope", batch=1, seq=64, heads=32, heads_k=8, dim=128, dtype="bf16", sections="16-24-24", interleaved=False, span=4096)
    return _named(name, c, kw)


def _write(name, **kw):
    """The same rotation while serving: q rotated, k rotated and put into the cache with v at the slot of each token."""
    c = dict(op="write", tokens=64, heads=32, heads_k=8, dim=128, dtype="bf16", sections="64", interleaved=False, span=4096, page=64,
             pages=64)
    return _named(name, c, kw)


def _plan(name, **kw):
    """Pages and slots for the new tokens of a batch: `nodes` > 0 drafted tokens for every sequence together with the
    tree's visibility words and positions, else ragged prompts of new_lo to new_hi tokens; then the pages go back."""
    c = dict(op="plan", batch=32, nodes=0, new_lo=1, new_hi=1, len_lo=0, len_hi=4096, page=64)
    return _named(name, c, kw)


def _keep(name, **kw):
    """After verification: the accepted path of every tree moves up behind the tokens before it, in all caches."""
    c = dict(op="keep", layers=1, batch=4, nodes=16, depth=4, heads_k=8, dim=128, dtype="bf16", len_lo=1, len_hi=100, page=64)
    return _named(name, c, kw)


def _named(name, c, kw):
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user, a short chain of drafts on a small model: launches and host time are what is waited for
        _tree("tree_one_user", batch=1, nodes=5, heads=16, heads_k=16, dim=64, len_lo=200, len_hi=200, append=True),
        # four drafts per sequence on a serving batch: 16 query rows per KV head, the cache's bytes count
        _tree("tree_few_drafts", batch=16, nodes=4, len_lo=1000, len_hi=8000, page=256),
        # odd sizes, ragged lengths from nothing on, a head dim between the kernels' own, small pages, tokens appended
        _tree("tree_ragged_odd", batch=13, nodes=27, heads=12, heads_k=2, dim=96, dtype="fp16", len_lo=0, len_hi=5000, page=64, append=True),
        # wide trees on a full batch: 256 query rows per KV head, where the cache's bytes and the products weigh alike
        _tree("tree_wide", batch=32, nodes=64, len_lo=8192, len_hi=16000, page=128),
        # a small training step on packed sequences, odd sizes, pairs next to each other
        _rope("axes_train_odd", batch=0, seq=777, heads=6, heads_k=2, dim=80, dtype="fp16", sections="8-16-16", interleaved=True, span=1500),
        # a training step on text with images: 32768 tokens, three axes
        _rope("axes_train", batch=8, seq=4096, span=8192),
        # one token for each of 64 sequences
        _write("write_tokens", tokens=64),
        # a chunk of prompts with images
        _write("write_prompts", tokens=8192, sections="16-24-24", pages=256, page=64, span=8192),
        # a step of drafted trees on a serving batch
        _plan("plan_trees", batch=64, nodes=32, len_lo=100, len_hi=8000, page=64),
        # a packed batch of prompts on top of what some of them have in the cache already
        _plan("plan_prompts", batch=256, new_lo=1, new_hi=2048, len_lo=0, len_hi=500, page=64),
        # one layer's caches, a few sequences
        _keep("keep_one_layer"),
        # all layers of a model on a serving batch
        _keep("keep_all_layers", layers=32, batch=64, nodes=64, depth=8, len_lo=10, len_hi=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "tree", "rope", "rope", "write", "write", "plan", "plan", "keep"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    heads_k = rng.choice([1, 2, 3, 4, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 6, 8])
    if op == "tree":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 160, 192, 256])
        batch = _log(rng, 1, 64)
        nodes = _log(rng, 1, 128)
        while batch * nodes * heads_k * group > 32 * 64 * 32:
            nodes = max(1, nodes // 2)
            group = 1 if nodes == 1 and group > 1 and batch * heads_k * group > 65536 else group
        most = 32 * 12000 * 8 * 128 // (batch * heads_k * dim)
        by_products = 32 * 64 * 32 * 12000 * 128 // (batch * nodes * heads_k * group * dim)
        hi = _log(rng, 1, max(2, min(16000, most, by_products)))
        small = batch * hi * heads_k * dim < 1 << 25
        return _tree("", batch=batch, nodes=nodes, heads=heads_k * group, heads_k=heads_k, dim=dim, dtype=dtype, len_lo=rng.choice([0, hi // 8, hi // 2, hi]),
                     len_hi=hi, page=rng.choice([0, 64, 64, 128, 256]), append=small and rng.random() < 0.5)
    if op in ("rope", "write"):
        dim = rng.choice([64, 72, 80, 96, 128, 128, 128, 192, 256])
        pairs = rng.choice([dim // 2, dim // 2, dim // 2, dim // 4, rng.randrange(3, dim // 2)])
        axes = rng.choice([1, 2, 3, 3, 4]) if pairs >= 8 else 1
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = "-".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))
        c = dict(heads=heads_k * group, heads_k=heads_k, dim=dim, dtype=dtype, sections=sections, interleaved=rng.random() < 0.4,
                 span=_log(rng, 1000, 16384))
        per_token = heads_k * (group + 2) * dim
        if op == "rope":
            batch = rng.choice([0, 1, 2, 5, 8])
            return _rope("", batch=batch, seq=_log(rng, 1, max(2, 8 * 4096 * 40 * 128 // (per_token * max(1, batch)) // 2)), **c)
        tokens = _log(rng, 1, max(2, min(16384, 8192 * 48 * 128 // per_token)))
        page = rng.choice([64, 128, 256])
        return _write("", tokens=tokens, page=page, pages=-(-tokens // page) + _log(rng, 1, 32), **c)
    if op == "plan":
        batch, page = _log(rng, 1, 512), rng.choice([16, 64, 64, 128, 256])
        if rng.random() < 0.5:
            return _plan("", batch=batch, nodes=_log(rng, 1, 128), len_lo=0, len_hi=_log(rng, 1, 16000), page=page)
        return _plan("", batch=batch, new_lo=0, new_hi=_log(rng, 1, 400000 // batch), len_lo=0, len_hi=_log(rng, 1, 2000), page=page)
    nodes = _log(rng, 2, 64)
    return _keep("", layers=rng.randrange(1, 16), batch=_log(rng, 1, 48), nodes=nodes, depth=rng.randrange(1, min(nodes, 12) + 1), heads_k=heads_k,
                 dim=rng.choice([64, 80, 128, 128, 256]) if heads_k <= 8 else 64, dtype=dtype, len_lo=0, len_hi=_log(rng, 1, 200), page=rng.choice([0, 64, 128]))


# ----------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 2 + 1)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _ints(g, lo, hi, shape, dtype=torch.int32):
    """Whole numbers from lo to hi, both among them."""
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV, dtype=dtype)


def _lengths(g, c):
    """Lengths of the sequences; one of them is the longest there is."""
    n = _ints(g, c["len_lo"], c["len_hi"], (c["batch"],))
    n[0] = c["len_hi"]
    return n


def _parents(g, batch, nodes):
    """Trees as a drafter makes them: node 0 hangs on the cache, every other one on an earlier node, near ones first."""
    i = torch.arange(nodes, device=DEV)
    back = 1 + (torch.rand((batch, nodes), generator=g, device=DEV) ** 2 * 6).long()
    return torch.where(i > 0, (i - back).clamp(min=0), i * 0 - 1).int()


def _ancestors(parents):
    """(batch, nodes, nodes): j is i or above it."""
    batch, nodes = parents.shape
    i = torch.arange(nodes, device=DEV)
    m = ((parents[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, math.ceil(math.log2(max(2, nodes))))):
        m = (m @ m > 0).float()
    return m > 0


def _words(mask):
    """32 flags to an int32, the first in the lowest bit."""
    nodes = mask.shape[-1]
    m = torch.nn.functional.pad(mask.long(), (0, -nodes % 32)).unflatten(-1, (-1, 32))
    w = (m << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _table(g, batch, per_seq, spare=3):
    """A page for every entry, in any order, in a pool with some spare ones."""
    pool = batch * per_seq + spare
    return torch.randperm(pool, generator=g, device=DEV)[: batch * per_seq].view(batch, per_seq).int(), pool


def _sections(c):
    return tuple(int(x) for x in c["sections"].split("-"))


def _positions(g, axes, tokens, span):
    """Stretches of 256 tokens: text, where all axes count alike, and images, where the first stands still and the others
    walk a grid 16 wide."""
    i = torch.arange(tokens, device=DEV)
    start = _ints(g, 0, max(0, span - 300), (tokens // 256 + 1,), torch.int64)[i // 256]
    r = i % 256
    image = (i // 256) % 2 == 1
    rows = [torch.where(image, start, start + r), torch.where(image, start + r // 16, start + r), torch.where(image, start + r % 16, start + r),
            start + r // 4]
    return torch.stack(rows[:axes]).clamp(max=span - 1).int().contiguous()


def _angle_tables(pairs, span, dtype):
    freq = 10000.0 ** (-torch.arange(pairs, device=DEV, dtype=torch.float64) / pairs)
    angle = torch.arange(span, device=DEV, dtype=torch.float64)[:, None] * freq
    return angle.cos().to(dtype), angle.sin().to(dtype)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"c": c}
    if c["op"] == "tree":
        dt, T, D = DTYPES[c["dtype"]], c["nodes"], c["dim"]
        most = c["len_hi"] + T
        if c["page"]:
            s["block_table"], pool = _table(g, c["batch"], -(-most // c["page"]))
            shape = (pool, c["page"], c["heads_k"], D)
        else:
            s["block_table"], shape = None, (c["batch"], most, c["heads_k"], D)
        s["k_cache"], s["v_cache"] = _normal(g, shape, dt), _normal(g, shape, dt)
        s["q"] = _normal(g, (c["batch"], T, c["heads"], D), dt)
        s["k"] = _normal(g, (c["batch"], T, c["heads_k"], D), dt) if c["append"] else None
        s["v"] = _normal(g, (c["batch"], T, c["heads_k"], D), dt) if c["append"] else None
        s["lens"] = _lengths(g, c)
        s["tree"] = _words(_ancestors(_parents(g, c["batch"], T)))
    elif c["op"] == "rope":
        dt, sec = DTYPES[c["dtype"]], _sections(c)
        tokens = max(1, c["batch"]) * c["seq"]
        lead = (c["batch"], c["seq"]) if c["batch"] else (c["seq"],)
        s["cos"], s["sin"] = _angle_tables(sum(sec), c["span"], dt)
        s["positions"] = _positions(g, len(sec), tokens, c["span"]).view((len(sec),) + lead)
        for name, h in (("q", c["heads"]), ("k", c["heads_k"]), ("dq", c["heads"]), ("dk", c["heads_k"])):
            s[name] = _normal(g, lead + (h, c["dim"]), dt)
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
    elif c["op"] == "write":
        dt, sec = DTYPES[c["dtype"]], _sections(c)
        s["cos"], s["sin"] = _angle_tables(sum(sec), c["span"], dt)
        s["positions"] = _positions(g, len(sec), c["tokens"], c["span"])
        for name, h in (("q", c["heads"]), ("k", c["heads_k"]), ("v", c["heads_k"])):
            s[name] = _normal(g, (c["tokens"], h, c["dim"]), dt)
        shape = (c["pages"], c["page"], c["heads_k"], c["dim"])
        s["k_cache"], s["v_cache"] = _normal(g, shape, dt), _normal(g, shape, dt)
        slots = torch.randperm(c["pages"] * c["page"], generator=g, device=DEV)[: c["tokens"]]
        # one token in about twenty is padding
        s["slots"] = torch.where(torch.rand(c["tokens"], generator=g, device=DEV) < 0.05, slots * 0 - 1, slots)
    elif c["op"] == "plan":
        B, ps = c["batch"], c["page"]
        s["lens"] = _lengths(g, c)
        # prompts of all lengths between the two, in any order; the packed batch is padded as a program does that keeps few sizes
        new = [c["nodes"] or c["new_lo"] + (c["new_hi"] - c["new_lo"]) * (2 * i + 1) // (2 * B) for i in range(B)]
        s["new"] = torch.tensor(new, dtype=torch.int32, device=DEV)[torch.randperm(B, generator=g, device=DEV)]
        s["total"] = sum(new) if c["nodes"] else -(-sum(new) // 64) * 64 + 64
        per_seq = -(-(c["len_hi"] + max(c["new_hi"], c["nodes"])) // ps)
        order = torch.randperm(2 * B * per_seq + 5, generator=g, device=DEV).int()
        s["block_table"] = order[: B * per_seq].view(B, per_seq).clone()
        s["free_pages"] = order[B * per_seq:].clone()
        # most of what may be asked for, so that the last requests may find the pool empty
        most = -(-max(c["new_hi"], c["nodes"]) // ps) + 1
        s["num_free"] = torch.tensor([max(1, min(int(B * most * 0.7) + 2, s["free_pages"].numel())), 0], dtype=torch.int32, device=DEV)
        s["parents"] = _parents(g, B, c["nodes"]) if c["nodes"] else None
    else:
        dt, T = DTYPES[c["dtype"]], c["nodes"]
        most = c["len_hi"] + T
        s["lens"] = _lengths(g, c)
        if c["page"]:
            s["block_table"], pool = _table(g, c["batch"], -(-most // c["page"]))
            shape = (pool, c["page"], c["heads_k"], c["dim"])
        else:
            s["block_table"], shape = None, (c["batch"], most, c["heads_k"], c["dim"])
        s["caches"] = torch.randint(-30000, 30000, (2 * c["layers"],) + shape, generator=g, device=DEV, dtype=torch.int16).to(dt)
        step = _ints(g, 1, max(1, (T - 1) // c["depth"]), (c["batch"], c["depth"]))
        step[:, 0] = 0
        i = torch.arange(c["depth"], device=DEV)
        count = _ints(g, 1, c["depth"], (c["batch"], 1))
        s["path"] = torch.where(i < count, step.cumsum(1).int(), -1).int()
    return s


# ----------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["c"]
    return (_RUN_OWN if own else _RUN_PLAIN)[c["op"]](s, c)


# The framework's calls
def _own_tree(s, c):
    from flash_attention_b200 import flash_attn_tree_with_kvcache

    out, lse = flash_attn_tree_with_kvcache(s["q"], s["k_cache"], s["v_cache"], s["tree"], s["lens"], k=s["k"], v=s["v"],
                                            block_table=s["block_table"], return_softmax_lse=True)
    return _tree_outputs(s, c, out, lse)


def _own_rope(s, c):
    from flash_attention_b200.layers.rotary import apply_rotary_emb_axes

    q, k = apply_rotary_emb_axes(s["q"], s["k"], s["cos"], s["sin"], s["positions"], _sections(c), interleaved=c["interleaved"])
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_write(s, c):
    from flash_attention_b200.layers.rotary import rotary_axes_to_cache

    q = rotary_axes_to_cache(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], _sections(c), s["slots"], s["k_cache"], s["v_cache"],
                             interleaved=c["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_plan(s, c):
    from flash_attention_b200 import paged_cache

    slots, positions, cu_seqlens, seqlens = paged_cache.reserve_pages(s["block_table"], s["lens"], s["new"], s["free_pages"], s["num_free"],
                                                                      c["page"], s["total"])
    left = s["num_free"].clone()
    tree = paged_cache.tree_layout(s["parents"], s["lens"]) if c["nodes"] else ()
    paged_cache.release_pages(s["block_table"], seqlens, s["lens"], s["free_pages"], s["num_free"], c["page"])
    return {"slots": slots, "positions": positions, "cu_seqlens": cu_seqlens, "seqlens": seqlens, "left": left, "tree": tree,
            "block_table": s["block_table"], "free_pages": s["free_pages"], "num_free": s["num_free"]}


def _own_keep(s, c):
    from flash_attention_b200 import paged_cache

    lens = paged_cache.keep_tree_path(s["caches"].unbind(0), s["lens"], s["path"], c["nodes"], block_table=s["block_table"])
    return {"caches": s["caches"], "lens": lens}


# The plain forms
def _tree_outputs(s, c, out, lse):
    r = {"out": out, "lse": lse}
    if c["append"]:
        r.update(k_cache=s["k_cache"], v_cache=s["v_cache"])
    return r


def _row_places(s, c, rows):
    """Places in the flat cache of rows (batch, n) of the sequences."""
    if s["block_table"] is None:
        return torch.arange(rows.shape[0], device=DEV)[:, None] * (c["len_hi"] + c["nodes"]) + rows
    return s["block_table"].long().gather(1, rows // c["page"]) * c["page"] + rows % c["page"]


def _plain_tree(s, c):
    B, T, Hk, D = c["batch"], c["nodes"], c["heads_k"], c["dim"]
    G, S = c["heads"] // Hk, c["len_hi"] + T
    lens = s["lens"].long()[:, None]
    if c["append"]:
        at = _row_places(s, c, lens + torch.arange(T, device=DEV))
        s["k_cache"].view(-1, Hk, D)[at] = s["k"]
        s["v_cache"].view(-1, Hk, D)[at] = s["v"]
    key = torch.arange(S, device=DEV)
    at = _row_places(s, c, key.expand(B, S))
    k, v = s["k_cache"].view(-1, Hk, D)[at].float(), s["v_cache"].view(-1, Hk, D)[at].float()
    q = s["q"].float().view(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    scores = (q @ k.permute(0, 2, 3, 1)).view(B, Hk, G, T, S).mul_(D ** -0.5)
    j = (key - lens).clamp(0, T - 1)  # node of a key
    bit = s["tree"].gather(2, (j // 32)[:, None].expand(B, T, S)) >> (j % 32)[:, None] & 1
    sees = (key < lens)[:, None] | (key < lens + T)[:, None] & (bit > 0)
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, Hk, G * T, S) @ v.transpose(1, 2)).view(B, Hk, G, T, D) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).reshape(B, T, c["heads"], D).to(s["q"].dtype)
    lse = torch.where(total > 0, total.log() + top, torch.full_like(top, math.inf)).view(B, c["heads"], T)
    return _tree_outputs(s, c, out, lse)


def _turned(x, cos, sin, interleaved):
    """Rows (tokens, heads, dim) by the angles (tokens, pairs), in 32 bits, rounded once."""
    pairs = cos.shape[-1]
    f = x.float()
    a, b = (f[..., 0:2 * pairs:2], f[..., 1:2 * pairs:2]) if interleaved else (f[..., :pairs], f[..., pairs:2 * pairs])
    cos, sin = cos[..., None, :], sin[..., None, :]
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, f[..., 2 * pairs:]), -1).to(x.dtype)


def _angles(s, c):
    """cos and sin of every token's pairs, each pair from the row of its axis."""
    sec = _sections(c)
    axis = torch.repeat_interleave(torch.arange(len(sec), device=DEV), torch.tensor(sec, device=DEV), output_size=sum(sec))
    row = s["positions"].long()[axis].movedim(0, -1)
    pair = torch.arange(sum(sec), device=DEV)
    return s["cos"].float()[row, pair], s["sin"].float()[row, pair]


def _plain_rope(s, c):
    cos, sin = _angles(s, c)
    turn = lambda name, way: _turned(s[name].detach(), cos, way * sin, c["interleaved"])  # noqa: E731
    return {"q": turn("q", 1), "k": turn("k", 1), "dq": turn("dq", -1), "dk": turn("dk", -1)}


def _plain_write(s, c):
    cos, sin = _angles(s, c)
    q, k = _turned(s["q"], cos, sin, c["interleaved"]), _turned(s["k"], cos, sin, c["interleaved"])
    real = s["slots"] >= 0
    at = s["slots"][real]
    s["k_cache"].view(-1, c["heads_k"], c["dim"])[at] = k[real]
    s["v_cache"].view(-1, c["heads_k"], c["dim"])[at] = s["v"][real]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_plan(s, c):
    ps, table, free = c["page"], s["block_table"], s["free_pages"]
    pages_of = lambda n: (n + ps - 1) // ps  # noqa: E731
    lens, new, num_free, per_seq = s["lens"].long(), s["new"].long(), s["num_free"][0].long(), table.shape[1]
    have, want = pages_of(lens), pages_of(lens + new)
    need = torch.where(want <= per_seq, want - have, 0)
    before = need.cumsum(0) - need
    granted = (want <= per_seq) & ((need == 0) | (before + need <= num_free))
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    col = torch.arange(per_seq, device=DEV)
    taken = granted[:, None] & (col >= have[:, None]) & (col < want[:, None])
    nth = before[:, None] + col - have[:, None]
    table.copy_(torch.where(taken, free[(num_free - 1 - nth).clamp(0, free.numel() - 1)], table))
    t = torch.arange(s["total"], device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=c["batch"] - 1)
    real = t < cu[-1]
    pos = torch.where(real, lens[b] + t - cu[b], 0)
    page = table.long()[b, (pos // ps).clamp(max=per_seq - 1)]
    slots = torch.where(real & granted[b], page * ps + pos % ps, -1)
    seqlens = torch.where(granted, lens + new, lens)
    used = torch.where(granted, need, 0).sum()
    s["num_free"][0] -= used.int()
    left = s["num_free"].clone()
    tree = ()
    if c["nodes"]:
        sees = _ancestors(s["parents"])
        tree = (_words(sees), (lens[:, None] + sees.sum(-1) - 1).int())
    # the pages go back
    back = (pages_of(seqlens) - have).clamp(min=0)
    first = back.cumsum(0) - back
    nth = first[:, None] + col - have[:, None]
    at = torch.where((col >= have[:, None]) & (col < pages_of(seqlens)[:, None]), left[0] + back.sum() - 1 - nth, free.numel())
    longer = torch.nn.functional.pad(free, (0, 1))
    longer[at.flatten()] = table.flatten()
    free.copy_(longer[:-1])
    s["num_free"][0] += back.sum().int()
    return {"slots": slots, "positions": pos.int(), "cu_seqlens": cu.int(), "seqlens": seqlens.int(), "left": left, "tree": tree,
            "block_table": table, "free_pages": free, "num_free": s["num_free"]}


def _plain_keep(s, c):
    path, lens = s["path"].long(), s["lens"].long()[:, None]
    on = path >= 0
    src = _row_places(s, c, lens + path.clamp(min=0))
    dst = _row_places(s, c, lens + torch.where(on, torch.arange(c["depth"], device=DEV), 0))
    flat = s["caches"].view(s["caches"].shape[0], -1, c["heads_k"], c["dim"])
    # (a row that is not on the path is written onto itself: to the first node, which stays where it is)
    flat[:, dst] = flat[:, torch.where(on, src, src[:, :1])]
    return {"caches": s["caches"], "lens": (lens[:, 0] + on.sum(1)).int()}


_RUN_OWN = {"tree": _own_tree, "rope": _own_rope, "write": _own_write, "plan": _own_plan, "keep": _own_keep}
_RUN_PLAIN = {"tree": _plain_tree, "rope": _plain_rope, "write": _plain_write, "plan": _plain_plan, "keep": _plain_keep}


# ----------------------------------------------------------------------------------------------- the work of a pass
def work(case):
    c = case
    size = 2
    if c["op"] == "tree":
        keys = c["batch"] * ((c["len_lo"] + c["len_hi"]) / 2 + c["nodes"])
        rows = c["batch"] * c["nodes"] * c["heads"]
        moved = keys * c["heads_k"] * c["dim"] * 2 * size + rows * c["dim"] * 2 * size + rows * 4
        moved += c["batch"] * c["nodes"] * -(-c["nodes"] // 32) * 4
        if c["append"]:  # read here, written there, instead of read there
            moved += c["batch"] * c["nodes"] * c["heads_k"] * c["dim"] * 2 * size
        mean = (c["len_lo"] + c["len_hi"]) / 2 + math.log2(c["nodes"] + 1)
        return {"bytes": moved, "flops": 4.0 * rows * mean * c["dim"]}
    if c["op"] in ("rope", "write"):
        sec = _sections(c)
        tokens = max(1, c["batch"]) * c["seq"] if c["op"] == "rope" else c["tokens"]
        # q and k forward and backward, or q, k and v once: read and written; of the tables what the tokens use, at most all
        rows = 2 * (c["heads"] + c["heads_k"]) if c["op"] == "rope" else c["heads"] + 2 * c["heads_k"]
        turned = 2 * (c["heads"] + c["heads_k"]) if c["op"] == "rope" else c["heads"] + c["heads_k"]
        tables = min(tokens, c["span"]) * sum(sec) * 2 * size
        return {"bytes": tokens * (rows * c["dim"] * 2 * size + len(sec) * 4 + (8 if c["op"] == "write" else 0)) + tables,
                "flops": 6.0 * tokens * turned * sum(sec)}
    if c["op"] == "plan":
        new = c["batch"] * (c["nodes"] or (c["new_lo"] + c["new_hi"]) / 2)
        words = c["batch"] * c["nodes"] * (-(-c["nodes"] // 32) * 4 + 8) if c["nodes"] else 0
        return {"bytes": new * 12 + c["batch"] * 28 + 6 * 4 * (new / c["page"] + c["batch"]) + words, "flops": new}
    moved = c["batch"] * (c["depth"] - 1) / 2 * c["heads_k"] * c["dim"] * size * 2 * 2 * c["layers"]
    return {"bytes": max(moved, 1.0) + c["batch"] * (8 + 4 * c["depth"]), "flops": 0}


# ----------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "plan":
        return None  # whole numbers
    if c["op"] == "tree":
        return _exact_tree(s, c)
    if c["op"] == "rope":
        return {n: _exact_turn(s, c, s[n].detach(), -1 if n[0] == "d" else 1) for n in ("q", "k", "dq", "dk")}
    if c["op"] == "write":
        k = _exact_turn(s, c, s["k"], 1)
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for i, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                kc[slot // c["page"], slot % c["page"]] = k[i]
                vc[slot // c["page"], slot % c["page"]] = s["v"][i].double()
        return {"q": _exact_turn(s, c, s["q"], 1), "k_cache": kc, "v_cache": vc}
    caches, lens = s["caches"], s["lens"].tolist()
    was = caches.clone()
    place = lambda b, row: (b, row) if s["block_table"] is None else (int(s["block_table"][b, row // c["page"]]), row % c["page"])  # noqa: E731
    for b, path in enumerate(s["path"].tolist()):
        for i, node in enumerate(n for n in path if n >= 0):
            (p0, r0), (p1, r1) = place(b, lens[b] + node), place(b, lens[b] + i)
            caches[:, p1, r1] = was[:, p0, r0]
    return {"caches": caches, "lens": None}


def _exact_tree(s, c):
    T, Hk, D, ps = c["nodes"], c["heads_k"], c["dim"], c["page"]
    G = c["heads"] // Hk
    outs, lses = [], []
    shift = torch.arange(32, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        if s["block_table"] is None:
            kc, vc = s["k_cache"][b], s["v_cache"][b]
        else:
            pages = s["block_table"][b].long()
            kc, vc = s["k_cache"][pages].flatten(0, 1), s["v_cache"][pages].flatten(0, 1)
        k, v = kc[: n + T].double(), vc[: n + T].double()
        if c["append"]:
            k[n:], v[n:] = s["k"][b].double(), s["v"][b].double()
        sees = torch.ones((T, n + T), dtype=torch.bool, device=DEV)
        sees[:, n:] = ((s["tree"][b].long()[:, :, None] >> shift) & 1).flatten(1)[:, :T] > 0
        q = s["q"][b].double().view(T, Hk, G, D)
        logits = torch.einsum("thgd,khd->hgtk", q, k) / math.sqrt(D)
        logits = torch.where(sees, logits, -math.inf)
        lse = torch.logsumexp(logits, -1)
        outs.append(torch.einsum("hgtk,khd->thgd", torch.exp(logits - lse[..., None]).nan_to_num(0.0), v).reshape(T, c["heads"], D))
        lses.append(torch.where(lse == -math.inf, math.inf, lse).reshape(c["heads"], T))
    r = {"out": torch.stack(outs), "lse": torch.stack(lses)}
    if c["append"]:
        for n, new in (("k_cache", s["k"]), ("v_cache", s["v"])):
            cache = s[n]
            for b, length in enumerate(s["lens"].tolist()):
                for i in range(T):
                    row = length + i
                    page = b if s["block_table"] is None else int(s["block_table"][b, row // ps])
                    cache[page, row % ps if ps else row] = new[b, i]
            r[n] = cache
    return r


def _exact_turn(s, c, x, way):
    sec = _sections(c)
    out = x.double().clone()
    first = 0
    for axis, n in enumerate(sec):
        at = s["positions"][axis].long()
        for i in range(first, first + n):
            i0, i1 = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + sum(sec))
            z = torch.complex(s["cos"][:, i].double(), way * s["sin"][:, i].double())[at][..., None]
            z = z * torch.complex(x[..., i0].double(), x[..., i1].double())
            out[..., i0], out[..., i1] = z.real, z.imag
        first += n
    return out
