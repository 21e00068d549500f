"""The operators of a speculative step over a paged cache held in 4 bits, as they are measured: real
calls over the sizes, layouts and types a program makes them with.

A small model drafts tokens after each sequence's last token, as a chain or as a tree; the model runs
over all of them at once, keeps the branch that its own probabilities accept, and draws one token
more. Each case is a dict of plain values with an "op":
  table   (cos, sin) of a range of positions, with frequencies scaled for a longer context
  rope    rows of q and k rotated at positions of their own (a tree's rows: by depth; prompts: in order)
  tree    attention of the drafted rows, which lie last in the cache, over their sequence's positions
          before them, their ancestors and themselves
  verify  from the rows' logits the branch that is accepted, and the next token, by given random numbers
  keep    the accepted rows moved together in the cache, all layers

The cache format. A row is the D values (64 or 128) of one position and kv head, K or V, in groups
of 32. A group's scale is an f16 of 8 significant bits; a code in [-7, 7] is held as code + 8 in 4 bits.
A page holds `page` positions; per kv head, in this order:
  K codes   [page][4][D / 32] words; word (l, g) of a row: dims 32 g + 8 l .. +8, lowest bits first
  V codes   [page / 8][D] words; word (b, d): positions 8 b .. +8 of dim d, lowest bits first
  K scales  [D / 32][page] f16
  V scales  [D / 32][page] f16

Verification. Row 0 of a sequence is its last token, already decided; the others are drafts, each with
a parent among the rows before it. At an accepted row with target probabilities p = softmax(logits /
temperature) its drafted children x are tried in order: without draft probabilities x is accepted where
u S < p(x), S what p leaves after the children rejected before it (a child whose token was already
rejected there is never accepted); with them (a chain, whose tokens were drawn from q) where u q(x) <
p(x). Where none is accepted the next token is drawn from p without the rejected ones, or from
max(p - q, 0) after a rejection by q: the lowest id whose running sum exceeds the given number times the
whole sum. At temperature 0 the child that holds the row's first largest logit is accepted, else that id
is the next token.

With `own` the calls go through the framework; without it the same is computed by elementary torch
operations, in 32 bits or, where a choice hangs on it or an angle is far, in 64. exact() computes it
in 64 bits, sequence by sequence.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 151936  # of the package's own model


# ---- the cases ------------------------------------------------------------------------------


def listed():
    return [
        # a program's start: the table of the package's own model at its usual context
        dict(name="table 4096 x 64", op="table", positions=4096, rotary=64, first=0, theta=1e6, scaling="none", factor=1.0),
        # a context stretched eightfold, wider heads
        dict(name="table 131072 x 128 turns", op="table", positions=131072, rotary=128, first=0, theta=5e5, scaling="turns", factor=8.0),
        # one chat's tree of 16 rows, the package's own model: launch latency
        dict(name="rope 16 rows f32", op="rope", heads=14, kv=2, d=64, rotary=64, layout="half", seqs=1, rows=16, spread=0, begin=777, tree=1, type="f32", out="f32"),
        # a batch of long prompts, wider heads of which half is rotated, neighbours as pairs
        dict(name="rope 32768 rows bf16", op="rope", heads=32, kv=8, d=128, rotary=64, layout="interleaved", seqs=8, rows=32768, spread=50, begin=0, tree=0, type="bf16", out="bf16"),
        # one chat of the package's own model with a chain of four drafts: latency
        dict(name="tree 1 x 5 at 517 f32", op="tree", heads=14, kv=2, d=64, page=64, seqs=1, rows=5, most=517, spread=0, branch=1, type="f32"),
        # a serving batch of it at full context, small trees
        dict(name="tree 16 x 16 at 2048 f32", op="tree", heads=14, kv=2, d=64, page=64, seqs=16, rows=16, most=2048, spread=40, branch=3, type="f32"),
        # long conversations, wide trees, wider heads
        dict(name="tree 8 x 64 at 8192 bf16", op="tree", heads=32, kv=8, d=128, page=64, seqs=8, rows=64, most=8192, spread=20, branch=4, type="bf16"),
        # one chat, greedy, a tree of the likeliest tokens
        dict(name="verify 1 x 16 greedy", op="verify", seqs=1, rows=16, spread=0, vocab=VOCAB, branch=3, draft=0, hot=0, type="f32"),
        # a batch of chains of four drafts drawn from a draft model
        dict(name="verify 16 x 5 drawn", op="verify", seqs=16, rows=5, spread=0, vocab=VOCAB, branch=1, draft=1, hot=100, type="f32"),
        # a large batch with trees, most of it sampling
        dict(name="verify 48 x 8 trees", op="verify", seqs=48, rows=8, spread=40, vocab=VOCAB, branch=3, draft=0, hot=80, type="f32"),
        # one chat's accepted rows, the package's own model's layers: latency
        dict(name="keep 1 x 16", op="keep", kv=2, d=64, page=64, layers=24, seqs=1, rows=16, spread=0, begin=1000),
        # a large batch of wide trees, wider heads
        dict(name="keep 64 x 32", op="keep", kv=8, d=128, page=64, layers=32, seqs=64, rows=32, spread=50, begin=100),
    ]


HEADS = [(14, 2, 64), (14, 2, 64), (8, 8, 64), (16, 2, 64), (12, 4, 64), (32, 8, 128), (28, 4, 128), (16, 1, 128), (8, 8, 128), (40, 8, 128)]
SCALINGS = ["none", "linear", "base", "turns", "log_turns"]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["table", "rope", "rope", "tree", "tree", "tree", "tree", "verify", "verify", "verify", "keep", "keep"])
    heads, kv, d = rng.choice(HEADS)
    page, spread = rng.choice([32, 64, 64, 128, 256]), rng.randint(0, 95)
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "table":
        rotary = 8 * rng.randint(1, 16)
        return dict(op=op, positions=_log(rng, 64, 131072 * 128 // rotary // 2 * 2), rotary=rotary, first=rng.choice([0, _log(rng, 1, 100000)]),
                    theta=float(rng.choice([10000, 500000, 1000000])), scaling=rng.choice(SCALINGS), factor=rng.uniform(1.0, 32.0))
    if op == "rope":  # at most the rows of eight long prompts
        seqs = _log(rng, 1, 64)
        rows = max(seqs, _log(rng, 1, 32768 * 40 * 128 * 2 // ((heads + kv) * d * 4)))
        return dict(op=op, heads=heads, kv=kv, d=d, rotary=rng.choice([d, d, d // 2, 8 * rng.randint(1, d // 8)]), layout=rng.choice(["half", "interleaved"]),
                    seqs=seqs, rows=rows, spread=spread, begin=rng.choice([0, _log(rng, 1, 8000)]), tree=int(rows <= 64 * seqs and rng.random() < 0.7),
                    type=kind, out=rng.choice(["f32", "f16", "bf16"]))
    if op == "tree":
        seqs, rows = _log(rng, 1, 64), _log(rng, 1, 64)
        room = 8 * 50 * 8192 * 32 * 128 // (seqs * rows * heads * d)  # the largest listed case's products
        held = 8 * 8192 * 8 * 128 // (seqs * kv * d)  # and its cache
        most = max(rows, _log(rng, rows, max(rows, min(131072, room, held))))
        return dict(op=op, heads=heads, kv=kv, d=d, page=page, seqs=seqs, rows=rows, most=most, spread=spread, branch=rng.choice([1, 2, 3, 5]), type=kind)
    if op == "verify":
        vocab = _log(rng, 1000, VOCAB)
        seqs = _log(rng, 1, 64)
        rows = _log(rng, 1, max(1, min(64, 48 * 6 * VOCAB // (seqs * vocab))))
        branch = rng.choice([1, 1, 2, 3, 5])
        return dict(op=op, seqs=seqs, rows=rows, spread=spread, vocab=vocab, branch=branch, draft=int(branch == 1 and rng.random() < 0.7),
                    hot=rng.choice([0, 50, 100, 100]), type=kind)
    seqs, rows, layers = _log(rng, 1, 64), _log(rng, 1, 64), rng.randint(1, 32)
    fits = max(1, int(6e8 / (layers * _page_bytes(kv, d, page) * seqs)) - _span(rows, page)) * page
    return dict(op=op, kv=kv, d=d, page=page, layers=layers, seqs=max(1, min(seqs, int(6e8 / (layers * _page_bytes(kv, d, page) * (1 + _span(rows, page)))))),
                rows=rows, spread=spread, begin=_log(rng, 1, min(4000, fits)))


def _shorter(c):
    """By what share of the longest each of the case's sequences is shorter: up to `spread` percent,
    the same for every seed, so that a case's outputs keep their shape."""
    g = torch.Generator().manual_seed(131 * c["seqs"] + c["spread"])
    u = torch.rand(c["seqs"], generator=g)
    u[0] = 0.0
    return u * (c["spread"] / 100.0)


def _split(c):
    """c["rows"] rows over the sequences, a row each at least."""
    w = 1.0 - _shorter(c)
    spare = c["rows"] - c["seqs"]
    n = [1 + int(spare * float(x) / float(w.sum())) for x in w]
    n[0] += c["rows"] - sum(n)
    return n


def _counts(c):
    """Rows of each sequence (c["rows"] of the first)."""
    return [max(1, int(round(c["rows"] * (1.0 - float(x))))) for x in _shorter(c)]


def _lengths(c):
    """Positions of each sequence, its drafted rows included."""
    return [max(n, int(round(c["most"] * (1.0 - float(x))))) for n, x in zip(_counts(c), _shorter(c))]


def _span(rows, page):
    """Pages that `rows` positions from anywhere in a page on may touch."""
    return (rows + page - 2) // page + 1


# ---- the cache's format in torch --------------------------------------------------------------


def _page_bytes(kv, d, page):
    return kv * page * (d + d // 8)


def _quantise(x):
    """Codes (float, -7..7) and scales of x [..., d], f32."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    s = (g.abs().amax(-1) * (1.0 / 7.0)).half()
    s = ((s.view(torch.int16) + 4) & -8).view(torch.float16).float()  # 8 significant bits, half up
    r = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    return torch.round(g * r[..., None]).clamp_(-7, 7), s


def _nibbles(b):
    """[..., 4] bytes of words -> [..., 8] codes, lowest bits first."""
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _words(u):
    """[..., 8] codes -> [..., 4] bytes of words."""
    u = u.to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _streams(pages, kv, d, page):
    """K codes, V codes, K scales, V scales of pages' bytes [..., page bytes], per kv head."""
    b = pages.unflatten(-1, (kv, page * (d + d // 8)))
    return b.split([page * d // 2, page * d // 2, page * d // 16, page * d // 16], -1)


def _unpack(pages, kv, d, page):
    """K and V as f32 [..., page, kv, d] of pages' bytes [..., page bytes]."""
    lead, groups = pages.shape[:-1], d // 32
    kc, vc, ks, vs = _streams(pages, kv, d, page)
    k = _nibbles(kc.reshape(*lead, kv, page, 4, groups, 4)).transpose(-3, -2).reshape(*lead, kv, page, groups, 32)
    v = _nibbles(vc.reshape(*lead, kv, page // 8, d, 4)).transpose(-2, -1).reshape(*lead, kv, page, groups, 32)
    scale = lambda s: s.contiguous().view(torch.float16).reshape(*lead, kv, groups, page).transpose(-2, -1).float()  # noqa: E731
    back = lambda u, s: ((u.float() - 8.0) * scale(s)[..., None]).flatten(-2).movedim(-3, -2)  # noqa: E731
    return back(k, ks), back(v, vs)


def _pack(k, v, kv, d, page):
    """Pages' bytes of K and V [n, kv, page, d]."""
    n, groups = k.shape[0], d // 32
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    kw = _words((kc + 8).reshape(n, kv, page, groups, 4, 8).transpose(3, 4)).reshape(n, kv, -1)
    vw = _words((vc + 8).reshape(n, kv, page // 8, 8, d).transpose(3, 4)).reshape(n, kv, -1)
    scale = lambda s: s.half().transpose(2, 3).contiguous().view(torch.uint8).reshape(n, kv, -1)  # noqa: E731
    return torch.cat([kw, vw, scale(ks), scale(vs)], -1).reshape(n, -1)


# ---- what a program has in hand --------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _rand(g, *shape):
    return torch.rand(*shape, device=DEV, generator=g)


def _u32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _offsets(n):
    return _u32([0] + list(torch.tensor(n).cumsum(0).tolist()))


class State:
    """What a program holds before a call; `handle` is its cache object, made when first needed."""

    handle = None


def _trees(n, branch, seed):
    """Parents (within the sequence) of n[s] rows of each sequence, and their depths: a row hangs on one of
    the `branch` rows before it that could still have a child; row 0 is the root, whose parent is none."""
    g = torch.Generator().manual_seed(seed + 3)
    parents, depths = [], []
    for rows in n:
        p, d = [-1], [0]
        back = torch.randint(1, branch + 1, (rows,), generator=g).tolist()
        for i in range(1, rows):
            p.append(max(0, i - back[i]))
            d.append(d[p[-1]] + 1)
        parents += p
        depths += d
    return _u32(parents), _u32(depths)


def _pages_for(s, c, seed, need):
    """A pool in which the sequences' pages lie in any order, and the table that finds them."""
    g = _gen(seed + 1)
    s.max_pages = max(need) + 1
    s.pages = sum(need) + 3
    order = torch.randperm(s.pages, generator=g, device=DEV).to(torch.int32)
    s.table = torch.full((c["seqs"], s.max_pages), -1, dtype=torch.int32, device=DEV)
    first = 0
    for i, n in enumerate(need):
        s.table[i, :n] = order[first:first + n]
        first += n


def _row_seq(n):
    return torch.repeat_interleave(torch.arange(len(n), device=DEV), torch.tensor(n, device=DEV))


def prepare(case, seed):
    c, s = case, State()
    s.c = c
    g = _gen(seed)
    if c["op"] == "table":
        # another seed: another part of the positions, and another base
        s.first = c["first"] + seed % 4096
        s.theta = c["theta"] * (1.0 + (seed % 977) / 4096.0)
    elif c["op"] == "rope":
        n = _split(c)
        s.n, s.starts = n, [c["begin"] + 3 * i if c["begin"] else 0 for i in range(c["seqs"])]
        s.offsets, s.begin, s.row_seq = _offsets(n), _u32(s.starts), _row_seq(n)
        s.depths = _trees(n, 3, seed)[1] if c["tree"] else None
        t = TYPES[c["type"]]
        s.q = _randn(g, c["rows"], c["heads"], c["d"]).to(t)
        s.k = _randn(g, c["rows"], c["kv"], c["d"]).to(t)
        last = max(a + b for a, b in zip(s.starts, n))
        freq = 1e6 ** (-torch.arange(0, c["rotary"], 2, device=DEV, dtype=torch.float64) / c["rotary"])
        angle = torch.arange(last, device=DEV, dtype=torch.float64)[:, None] * freq
        s.table = torch.stack([angle.cos(), angle.sin()], -1).float()  # [positions][rotary / 2] (cos, sin)
    elif c["op"] == "tree":
        s.n, s.lens = _counts(c), _lengths(c)
        s.offsets, s.lengths = _offsets(s.n), _u32(s.lens)
        s.parents = _trees(s.n, c["branch"], seed)[0] if c["branch"] > 1 else None
        page = c["page"]
        _pages_for(s, c, seed, [-(-x // page) for x in s.lens])
        h = _gen(seed + 2)
        s.pool = torch.empty(s.pages, _page_bytes(c["kv"], c["d"], page), dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 27) // (c["kv"] * page * c["d"]))
        for at in range(0, s.pages, step):  # a part at a time, so that the values fit
            m = min(step, s.pages - at)
            s.pool[at:at + m] = _pack(*(_randn(h, m, c["kv"], page, c["d"]) for _ in range(2)), c["kv"], c["d"], page)
        s.q = _randn(g, sum(s.n), c["heads"], c["d"]).to(TYPES[c["type"]])
    elif c["op"] == "verify":
        s.n = _counts(c)
        rows, vocab = sum(s.n), c["vocab"]
        s.offsets, s.row_seq = _offsets(s.n), _row_seq(s.n)
        s.parents = _trees(s.n, c["branch"], seed)[0] if c["branch"] > 1 else None
        # a few likely tokens, a long tail; the draft model's view of it is the same, blurred
        logits = _randn(g, rows, vocab) * 2.0
        logits.scatter_add_(1, torch.randint(0, vocab, (rows, 8), device=DEV, generator=g), 10.0 + 8.0 * _rand(g, rows, 8))
        s.logits = logits.to(TYPES[c["type"]])
        blurred = logits.add_(_randn(g, rows, vocab) * 0.5)
        up = _up(s)
        if c["draft"]:
            s.draft = torch.softmax(blurred, -1)
            pick = (blurred - torch.log(-torch.log(_rand(g, rows, vocab).clamp_(1e-20, 1.0 - 1e-7)))).argmax(-1)
            s.tokens = pick[up].to(torch.int32)
        else:
            s.draft = None
            row = torch.arange(rows, device=DEV)
            siblings = (up[:, None] == up) & (row > up) & (row < row[:, None])  # those before a row
            rank = siblings.sum(-1).clamp(max=min(64, vocab) - 1)
            s.tokens = blurred.topk(min(64, vocab), -1).indices[up].gather(1, rank[:, None])[:, 0].to(torch.int32)
        s.accept = _rand(g, rows)
        s.draws = _rand(g, c["seqs"])
        s.temperatures = None
        if c["hot"]:
            warm = (torch.arange(c["seqs"], device=DEV) * 37 % 100) < c["hot"]  # the others greedy
            s.temperatures = torch.where(warm, 0.7 + 0.5 * _rand(g, c["seqs"]), torch.zeros(c["seqs"], device=DEV))
    else:
        s.n = _counts(c)
        s.lens = [c["begin"] + 5 * i % 64 + n for i, n in enumerate(s.n)]
        s.offsets, s.lengths = _offsets(s.n), _u32(s.lens)
        page, most = c["page"], max(s.n)
        _pages_for(s, c, seed, [(x - n) // page + _span(most, page) for x, n in zip(s.lens, s.n)])
        s.pool = torch.randint(0, 256, (s.pages, c["layers"] * _page_bytes(c["kv"], c["d"], page)), dtype=torch.uint8, device=DEV, generator=g)
        # each sequence keeps its row 0 and some of the others, in their order
        kept = torch.rand(c["seqs"], most, generator=torch.Generator().manual_seed(seed + 4)) < 0.4
        kept[:, 0] = True
        paths = [[j for j in range(n) if kept[i, j]] for i, n in enumerate(s.n)]
        s.counts = _u32([len(p) for p in paths])
        s.path = _u32([p + [-1] * (most - len(p)) for p in paths])
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------------------

_device = None


def _dev():
    global _device
    from enargeia_amd import kernels

    if _device is None:
        _device = kernels.Device(0)
    return _device


def _cache(s):
    """The cache object over the program's pool."""
    from enargeia_amd import kv4

    if s.handle is None:
        c = s.c
        s.handle = kv4.Kv4Cache(_dev(), kv_heads=c["kv"], head_dim=c["d"], page_size=c["page"], pages=s.pool.shape[0],
                                layers=c.get("layers", 1), pool=s.pool)
    return s.handle


def _run_own(s):
    from enargeia_amd import drafts

    c = s.c
    new = lambda *shape, t: torch.empty(*shape, dtype=t, device=DEV)  # noqa: E731
    if c["op"] == "table":
        table = new(c["positions"], c["rotary"] // 2, 2, t=torch.float32)
        drafts.rope_table(_dev(), table, positions=c["positions"], rotary_dim=c["rotary"], first=s.first, theta=s.theta,
                          scaling=c["scaling"], factor=c["factor"], context=8192, low=1.0, high=4.0, amplitude=_amplitude(c))
        return table
    if c["op"] == "rope":
        q, k = (new(*x.shape, t=TYPES[c["out"]]) for x in (s.q, s.k))
        drafts.rope(_dev(), s.table, rows=c["rows"], head_dim=c["d"], rotary_dim=c["rotary"], table_positions=s.table.shape[0],
                    q=s.q, q_out=q, heads=c["heads"], k=s.k, k_out=k, kv_heads=c["kv"], positions=s.depths, offsets=s.offsets,
                    starts=s.begin, sequences=c["seqs"], layout=c["layout"], in_type=c["type"], out_type=c["out"])
        return {"q": q, "k": k}
    if c["op"] == "tree":
        out = new(*s.q.shape, t=s.q.dtype)
        _cache(s).attend_tree(s.q, s.offsets, s.lengths, s.table, out, parents=s.parents, heads=c["heads"], rows=s.q.shape[0],
                              max_rows=max(s.n), sequences=c["seqs"], max_pages=s.max_pages, type=c["type"])
        return out
    if c["op"] == "verify":
        path = new(c["seqs"], max(s.n), t=torch.int32)
        counts, token = (new(c["seqs"], t=torch.int32) for _ in range(2))
        drafts.verify(_dev(), s.logits, s.tokens, s.offsets, path, counts, token, parents=s.parents, draft=s.draft, accept=s.accept,
                      draws=s.draws, temperatures=s.temperatures, sequences=c["seqs"], rows=s.logits.shape[0], max_rows=max(s.n),
                      vocab=c["vocab"], type=c["type"])
        return {"path": path, "counts": counts, "next": token}
    lengths = new(c["seqs"], t=torch.int32)
    _cache(s).keep(s.path, s.counts, s.offsets, s.lengths, s.table, lengths, max_rows=max(s.n), sequences=c["seqs"], max_pages=s.max_pages)
    return {"pool": s.pool, "lengths": lengths}


def _amplitude(c):
    return 1.0 if c["scaling"] == "none" else 1.0 + 0.1 * math.log(c["factor"])


def _frequencies(c, theta):
    """Of the pairs of a rotated part, f64."""
    r, i = c["rotary"], torch.arange(0, c["rotary"], 2, device=DEV, dtype=torch.float64)
    if c["scaling"] == "base":  # the longest wave is stretched by the factor
        theta = theta * c["factor"] ** (r / (r - 2))
    f = theta ** (-i / r)
    if c["scaling"] == "linear":
        return f / c["factor"]
    if c["scaling"] in ("turns", "log_turns"):  # waves that turn 4 times and more in 8192 positions stay, under once are stretched
        turns = 8192.0 * f / (2.0 * math.pi)
        w = (turns - 1.0) / 3.0 if c["scaling"] == "turns" else torch.log(turns) / math.log(4.0)
        w = w.clamp(0.0, 1.0)
        return f * (w + (1.0 - w) / c["factor"])
    return f


def _positions(s):
    i = torch.arange(s.row_seq.numel(), device=DEV)
    within = i - s.offsets.long()[s.row_seq] if s.depths is None else s.depths.long()
    return s.begin.long()[s.row_seq] + within


def _rotate(x, cs, c):
    """x [rows, heads, d] (f32) with its first `rotary` dims turned by the rows' (cos, sin)."""
    r, co, si = c["rotary"], cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if c["layout"] == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    a, b = a * co - b * si, b * co + a * si
    t = torch.cat([a, b], -1) if c["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([t, x[..., r:]], -1)


def _grid(offsets, most):
    """Packed rows as [sequence, most]: which row, and whether there is one."""
    at = offsets[:-1, None].long() + torch.arange(most, device=DEV)
    have = at < offsets[1:, None]
    return torch.where(have, at, 0), have


def _ancestors(parents, offsets, most):
    """[sequence, most, most]: whether row j is row i or above it."""
    at, have = _grid(offsets, most)
    i = torch.arange(most, device=DEV)
    p = parents[at] if parents is not None else (i - 1).expand_as(at)
    step = ((p[..., None] == i) & have[..., None]).double() + torch.eye(most, device=DEV, dtype=torch.float64)
    return torch.matrix_power(step, most) > 0


def _up(s):
    """Each packed row's parent among all rows (of a root: itself)."""
    first = s.offsets.long()[s.row_seq]
    local = torch.arange(s.row_seq.numel(), device=DEV) - first
    p = local - 1 if s.parents is None else s.parents.long()
    return torch.where(local > 0, first + p, first)


def _run_plain(s):
    c = s.c
    if c["op"] == "table":
        p = torch.arange(c["positions"], device=DEV, dtype=torch.float64) + s.first
        angle = p[:, None] * _frequencies(c, s.theta)
        return (torch.stack([angle.cos(), angle.sin()], -1) * _amplitude(c)).float()
    if c["op"] == "rope":
        cs = s.table[_positions(s)]
        return {"q": _rotate(s.q.float(), cs, c).to(TYPES[c["out"]]), "k": _rotate(s.k.float(), cs, c).to(TYPES[c["out"]])}
    if c["op"] == "tree":
        n, kv, d, most = c["seqs"], c["kv"], c["d"], max(s.n)
        k, v = _unpack(s.pool[s.table.long().clamp(min=0)], kv, d, c["page"])  # [seqs, pages, page, kv, d]
        k, v = (x.reshape(n, -1, kv, d).transpose(1, 2) for x in (k, v))
        at, have = _grid(s.offsets, most)
        q = s.q.float()[at].reshape(n, most, kv, -1, d).permute(0, 2, 1, 3, 4)  # [seqs, kv, rows, group, d]
        group = q.shape[3]
        w = (q.reshape(n, kv, most * group, d) @ k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(d))
        rel = torch.arange(k.shape[2], device=DEV) - (s.lengths.long() - have.sum(-1))[:, None]  # position less the first drafted one
        seen = _ancestors(s.parents, s.offsets, most).gather(2, rel.clamp(0, most - 1)[:, None].expand(n, most, -1))
        seen = (rel < 0)[:, None] | (seen & (rel < have.sum(-1)[:, None])[:, None])
        w = w.masked_fill_(~seen[:, None, :, None].expand(n, 1, most, group, -1).reshape(n, 1, most * group, -1), -math.inf)
        w = w.sub_(w.amax(-1, keepdim=True)).exp_()
        o = ((w @ v) / w.sum(-1, keepdim=True)).reshape(n, kv, most, group, d).permute(0, 2, 1, 3, 4).reshape(n, most, c["heads"], d)
        return o[have].to(s.q.dtype)
    if c["op"] == "verify":
        return _verify_plain(s)
    kv, d, page, most = c["kv"], c["d"], c["page"], max(s.n)
    first = (s.lengths.long() - s.offsets.long().diff()) % page  # the first drafted slot in the window of pages
    i = torch.arange(most, device=DEV)
    moved = i < s.counts[:, None]
    span = _span(most, page)
    ids = s.table.long().gather(1, ((s.lengths.long() - s.offsets.long().diff()) // page)[:, None] + torch.arange(span, device=DEV))
    slots = torch.arange(span * page, device=DEV).repeat(c["seqs"], 1)
    source = slots.scatter(1, first[:, None] + i, torch.where(moved, first[:, None] + s.path, first[:, None] + i))
    b = s.pool[ids].unflatten(-1, (c["layers"], -1))  # [seqs, span, layers, page bytes]
    kc, vc, ks, vs = (x.movedim(1, 3) for x in _streams(b, kv, d, page))  # [seqs, layers, kv, span, ...]
    lead, groups = kc.shape[:3], d // 32
    pick = lambda x: x.gather(3, source[:, None, None, :, None].expand(*lead, -1, x.shape[-1]))  # noqa: E731 (slots along 3)
    by_slot = lambda x: x.reshape(*lead, span, groups, page, 2).transpose(4, 5).reshape(*lead, span * page, -1)  # noqa: E731
    off = lambda x: x.reshape(*lead, span, page, groups, 2).transpose(4, 5).reshape(*lead, span, -1)  # noqa: E731
    v = _nibbles(vc.reshape(*lead, span, page // 8, d, 4)).transpose(-2, -1).reshape(*lead, span * page, d)
    v = pick(v).reshape(*lead, span, page // 8, 8, d).transpose(-2, -1)
    new = [pick(kc.reshape(*lead, span * page, d // 2)).reshape(*lead, span, -1), _words(v).reshape(*lead, span, -1), off(pick(by_slot(ks))), off(pick(by_slot(vs)))]
    s.pool[ids] = torch.cat(new, -1).movedim(3, 1).reshape(c["seqs"], span, -1)
    return {"pool": s.pool, "lengths": (s.lengths - s.offsets.diff() + s.counts).int()}


def _verify_plain(s):
    c, n = s.c, s.row_seq.numel()
    most, vocab = max(s.n), c["vocab"]
    up, tokens, root = _up(s), s.tokens.long(), s.offsets.long()[s.row_seq]
    row = torch.arange(n, device=DEV)
    temperature = torch.zeros(c["seqs"], device=DEV, dtype=torch.float64) if s.temperatures is None else s.temperatures.double()
    greedy = temperature == 0.0
    x = s.logits.double()
    top = x.amax(-1, keepdim=True)
    best = torch.where(x == top, torch.arange(vocab, device=DEV), vocab).amin(-1)
    e = torch.exp((x - top) / torch.where(greedy, 1.0, temperature)[s.row_seq][:, None])
    p = e / e.sum(-1, keepdim=True)
    px = p[up, tokens]  # of a row's token where it was drafted
    siblings = (up[:, None] == up[None, :]) & (row > root) & (row < row[:, None])  # those before a row
    same = siblings & (tokens[:, None] == tokens[None, :])
    fresh = ~same.any(-1)  # (a token that a sibling had before is not counted again)
    if s.draft is None:
        left = 1.0 - (siblings & fresh).double() @ px
        ok = (s.accept.double() * left < px) & fresh
    else:
        ok = s.accept.double() * s.draft.double()[up, tokens] < px
    ok = torch.where(greedy[s.row_seq], tokens == best[up], ok) & (row > root)
    chosen = ok & ~(siblings & ok).any(-1)  # the first of its siblings that passes
    at, have = _grid(s.offsets, most)
    above = _ancestors(s.parents, s.offsets, most)
    fine = (chosen | (row == root))[at] & have
    taken = fine & ~(above & ~fine[:, None, :]).any(-1)
    counts = taken.sum(-1)
    path = torch.where(taken, torch.arange(most, device=DEV), most).sort(-1).values
    last = at.gather(1, path.gather(1, counts[:, None] - 1))[:, 0]
    mass = p[last]
    tried = (up[None, :] == last[:, None]) & (row > root)  # the last accepted row's children, all rejected
    if s.draft is None:
        gone = torch.zeros(c["seqs"], vocab, device=DEV, dtype=torch.float64).index_put_(
            (tried.nonzero()[:, 0], tokens[tried.nonzero()[:, 1]]), torch.ones((), device=DEV, dtype=torch.float64), accumulate=True)
        mass = torch.where(gone > 0, 0.0, mass)
    else:
        mass = torch.where(tried.any(-1)[:, None], (mass - s.draft[last].double()).clamp(min=0.0), mass)
    running = mass.cumsum(-1)
    drawn = (running <= s.draws.double()[:, None] * running[:, -1:]).sum(-1).clamp(max=vocab - 1)
    token = torch.where(greedy, best[last], drawn)
    path = torch.where(torch.arange(most, device=DEV) < counts[:, None], path, -1)
    return {"path": path.int(), "counts": counts.int(), "next": token.int()}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "table":
        return {"bytes": c["positions"] * c["rotary"] * 4, "flops": c["positions"] * c["rotary"] * 2}
    if c["op"] == "rope":
        width = (c["heads"] + c["kv"]) * c["d"]
        return {"bytes": c["rows"] * (width * (SIZE[c["type"]] + SIZE[c["out"]]) + 4 * c["rotary"]),
                "flops": 3 * c["rows"] * (c["heads"] + c["kv"]) * c["rotary"]}
    n = _counts(c)
    if c["op"] == "tree":
        held = 2 * c["kv"] * (c["d"] // 2 + c["d"] // 16)  # of one position
        pairs = sum(r * (x - r) + r for r, x in zip(n, _lengths(c)))  # (and a few ancestors)
        return {"bytes": sum(_lengths(c)) * held + 2 * sum(n) * c["heads"] * c["d"] * SIZE[c["type"]],
                "flops": 4 * c["d"] * c["heads"] * pairs}
    if c["op"] == "verify":  # all rows' logits, and the row of the draft's probabilities where the branch ends
        values = sum(n) * c["vocab"]
        return {"bytes": values * SIZE[c["type"]] + (c["seqs"] * c["vocab"] * 4 if c["draft"] else 0), "flops": 4 * values}
    held = 2 * c["layers"] * c["kv"] * (c["d"] // 2 + c["d"] // 16)
    return {"bytes": max(1, int(2 * 0.4 * sum(n) * held)), "flops": 0}  # (the rows that move, about)


# ---- the definition in 64 bits, sequence by sequence -------------------------------------------


def _code64(words, i):
    return ((words.long() >> (4 * i)) & 15).double() - 8.0


def _row64(s, seq, upto):
    """K and V [upto, kv, d] of a sequence in 64 bits, from its pages word by word."""
    c = s.c
    page, d, kv = c["page"], c["d"], c["kv"]
    ids = s.table[seq, : -(-upto // page)].long()
    b = s.pool[ids].reshape(len(ids), kv, -1)
    half = page * d // 2
    kw, vw = (b[..., i * half:(i + 1) * half].contiguous().view(torch.int32).long() & 0xFFFFFFFF for i in range(2))
    ks, vs = b[..., 2 * half:].contiguous().view(torch.float16).double().reshape(len(ids), kv, 2, d // 32, page).unbind(2)
    k = torch.empty(len(ids), kv, page, d, dtype=torch.float64, device=DEV)
    v = torch.empty_like(k)
    kw, vw = kw.reshape(len(ids), kv, page, 4, d // 32), vw.reshape(len(ids), kv, page // 8, d)
    for grp in range(d // 32):
        for part in range(4):
            for i in range(8):
                at = 32 * grp + 8 * part + i
                k[..., at] = _code64(kw[..., part, grp], i) * ks[:, :, grp]
    for i in range(8):
        v[:, :, i::8] = _code64(vw, i)
    v *= vs.repeat_interleave(32, 2).transpose(2, 3)
    return tuple(x.transpose(1, 2).reshape(-1, kv, d)[:upto] for x in (k, v))


def _turn64(x, angle_cs, c):
    """Rows x [n, heads, d] turned as complex numbers."""
    y, r = x.double().clone(), c["rotary"]
    z = torch.view_as_complex(angle_cs.double().contiguous())[:, None]
    first, second = (slice(0, r // 2), slice(r // 2, r)) if c["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    t = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = t.real, t.imag
    return y


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "table":
        out = torch.empty(c["positions"], c["rotary"] // 2, 2, dtype=torch.float64, device=DEV)
        p = s.first + torch.arange(c["positions"], device=DEV, dtype=torch.float64)
        for i in range(c["rotary"] // 2):  # a pair at a time, its frequency in Python's numbers
            base = s.theta * c["factor"] ** (c["rotary"] / (c["rotary"] - 2)) if c["scaling"] == "base" else s.theta
            f = math.exp(-2.0 * i / c["rotary"] * math.log(base))
            if c["scaling"] == "linear":
                f /= c["factor"]
            elif c["scaling"] in ("turns", "log_turns"):
                turns = 8192.0 * f / (2.0 * math.pi)
                w = (turns - 1.0) / 3.0 if c["scaling"] == "turns" else math.log(turns, 4.0)
                w = min(1.0, max(0.0, w))
                f = w * f + (1.0 - w) * f / c["factor"]
            z = torch.polar(torch.full_like(p, _amplitude(c)), p * f)
            out[:, i, 0], out[:, i, 1] = z.real, z.imag
        return out
    if c["op"] == "rope":
        outs, at = {"q": [], "k": []}, 0
        for n, start in zip(s.n, s.starts):
            rows = slice(at, at + n)
            p = start + (s.depths[rows].long() if s.depths is not None else torch.arange(n, device=DEV))
            for name, x in (("q", s.q), ("k", s.k)):
                outs[name].append(_turn64(x[rows], s.table[p], c))
            at += n
        return {name: torch.cat(x) for name, x in outs.items()}
    if c["op"] == "tree":
        out = torch.empty(s.q.shape, dtype=torch.float64, device=DEV)
        r0 = 0
        for i, (n, length) in enumerate(zip(s.n, s.lens)):
            k, v = _row64(s, i, length)
            seen = torch.zeros(n, length, dtype=torch.bool)
            seen[:, : length - n] = True
            above = s.parents[r0:r0 + n].tolist() if s.parents is not None else list(range(-1, n - 1))
            for r in range(n):
                a = r
                while a >= 0:
                    seen[r, length - n + a] = True
                    a = above[a]
            seen = seen.to(DEV)
            for h in range(c["heads"]):
                j = h // (c["heads"] // c["kv"])
                w = s.q[r0:r0 + n, h].double() @ k[:, j].t().contiguous() / math.sqrt(c["d"])
                out[r0:r0 + n, h] = torch.softmax(w.masked_fill(~seen, -math.inf), -1) @ v[:, j].contiguous()
            r0 += n
        return out
    return None
