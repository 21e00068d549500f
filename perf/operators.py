"""The operators that serve several sequences over a paged cache held in 4 bits, as they are
measured: real calls over the sizes, layouts and types a program makes them with.

Each case is a dict of plain values with an "op":
  append  new rows of a batch: RoPE on q and k, k and v into the cache's pages (and read back, so
          that what the cache then holds is seen as values)
  read    cached rows of a batch as packed keys and values (what a later prompt chunk attends to)
  decode  attention of one token per sequence over the cache
  packed  causal attention over packed prompts of different lengths
  copy    pages copied over all layers (the tail page of a fork; a compaction)

The cache format. A row is the D values (64 or 128) of one position and kv head, K or V, in groups
of 32. A group's scale is absmax / 7 as f16, rounded to 8 significant bits (so that every value is
exact in f16); a code is round(x / scale) in [-7, 7], held as code + 8 in 4 bits. A page holds
`page` positions; per kv head, in this order:
  K codes   [page][4][D / 32] words; word (l, g) of a row: dims 32 g + 8 l .. +8, lowest bits first
  V codes   [page / 8][D] words; word (b, d): positions 8 b .. +8 of dim d, lowest bits first
  K scales  [D / 32][page] f16
  V scales  [D / 32][page] f16

With `own` the calls go through the framework; without it the same is computed by elementary torch
operations in 32 bits. exact() computes it in 64 bits, sequence by sequence.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
MOST_SCALE = 9344.0  # the largest scale whose codes stay finite in f16


# ---- the cases ------------------------------------------------------------------------------


def listed():
    return [
        # one token of one sequence of the package's own model: a decode step's append, launch latency
        dict(name="append 1 row f32", op="append", heads=14, kv=2, d=64, page=64, seqs=1, rows=1, begin=777, spread=0, type="f32", out="f32"),
        # eight prompts of different lengths, packed, as the prompt GEMM leaves them
        dict(name="append 16384 rows f32 to f16", op="append", heads=14, kv=2, d=64, page=64, seqs=8, rows=16384, begin=0, spread=50, type="f32", out="f16"),
        # the rows before a short prompt chunk of one sequence
        dict(name="read 1 x 500 f16", op="read", kv=2, d=64, page=32, seqs=1, rows=500, begin=0, spread=0, out="f16"),
        # long conversations that go on: all their rows, wider heads
        dict(name="read 16 x 4096 bf16", op="read", kv=8, d=128, page=64, seqs=16, rows=65536, begin=0, spread=30, out="bf16"),
        # one chat of the package's own model, one token: latency
        dict(name="decode 1 x 517 f32", op="decode", heads=14, kv=2, d=64, page=64, seqs=1, most=517, spread=0, type="f32"),
        # a serving batch of it at full context
        dict(name="decode 48 x 2048 f32", op="decode", heads=14, kv=2, d=64, page=64, seqs=48, most=2048, spread=60, type="f32"),
        # a large batch of long sequences, wider heads
        dict(name="decode 32 x 16384 bf16", op="decode", heads=32, kv=8, d=128, page=64, seqs=32, most=16384, spread=30, type="bf16"),
        # three short prompts
        dict(name="packed 3 x 150 f16", op="packed", heads=14, kv=2, d=64, seqs=3, most=150, spread=70, before=0, type="f16"),
        # a batch of ordinary prompts of the package's own model
        dict(name="packed 8 x 2048 f16", op="packed", heads=14, kv=2, d=64, seqs=8, most=2048, spread=60, before=0, type="f16"),
        # a long prompt, wider heads
        dict(name="packed 1 x 8192 bf16", op="packed", heads=32, kv=8, d=128, seqs=1, most=8192, spread=0, before=0, type="bf16"),
        # a conversation forked: its tail page copied, 24 layers a page
        dict(name="copy 1 page", op="copy", kv=2, d=64, page=64, layers=24, pages=64, count=1),
        # a cache compacted: half its pages move
        dict(name="copy 2000 pages", op="copy", kv=2, d=64, page=64, layers=24, pages=4096, count=2000),
    ]


HEADS = [(14, 2, 64), (14, 2, 64), (8, 8, 64), (16, 2, 64), (12, 4, 64), (32, 8, 128), (28, 4, 128), (16, 1, 128), (8, 8, 128), (40, 8, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "decode", "decode", "decode", "packed", "packed", "packed", "copy"])
    heads, kv, d = rng.choice(HEADS)
    page, spread = rng.choice([32, 64, 64, 128, 256]), rng.randint(0, 95)
    # (decode reaches from one position to a few very long documents, one kv head for many query heads)
    seqs = _log(rng, 1, 64)
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "append":  # at most the rows of eight long prompts
        rows = max(seqs, _log(rng, 1, 16384 * 64 * 14 // (heads * d)))
        return dict(op=op, heads=heads, kv=kv, d=d, page=page, seqs=seqs, rows=rows, begin=rng.choice([0, _log(rng, 1, 8000)]),
                    spread=spread, type=kind, out=rng.choice(["f32", "f16", "bf16"]))
    if op == "read":
        return dict(op=op, kv=kv, d=d, page=page, seqs=seqs, rows=max(seqs, _log(rng, 1, 65536 * 8 * 128 // (kv * d * 2))),
                    begin=rng.choice([0, _log(rng, 1, 8000)]), spread=spread, out=rng.choice(["f32", "f16", "bf16"]))
    if op == "decode":
        most = _log(rng, 1, min(131072, 32 * 16384 * 4 * 64 // (seqs * kv * d) * 2))
        return dict(op=op, heads=heads, kv=kv, d=d, page=page, seqs=seqs, most=most, spread=spread, type=kind)
    if op == "packed":
        seqs = _log(rng, 1, 24)
        most = _log(rng, 1, int(math.sqrt(6000 * 6000 * 32 * 128 / (seqs * heads * d))))
        return dict(op=op, heads=heads, kv=kv, d=d, seqs=seqs, most=min(most, 6000), spread=spread,
                    before=rng.choice([0, 0, _log(rng, 1, 2000)]), type=rng.choice(["f16", "bf16"]))
    layers = rng.randint(1, 24)
    pages = _log(rng, 4, min(8192, max(4, int(9e8 / (layers * _page_bytes(kv, d, page))))))
    return dict(op="copy", kv=kv, d=d, page=page, layers=layers, pages=pages, count=max(1, int(pages * rng.uniform(0.02, 0.48))))


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
    return [max(1, int(round(c["most"] * (1.0 - float(x))))) for x in _shorter(c)]


# ---- the cache's format in torch --------------------------------------------------------------


def _page_bytes(kv, d, page):
    return kv * page * (d + d // 8)


def _quantise(x):
    """Codes (float, -7..7) and scales of x [..., d], f32."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    a = g.abs().amax(-1)
    s = (a * (1.0 / 7.0)).clamp(max=MOST_SCALE).half()
    s = ((s.view(torch.int16) + 4) & -8).view(torch.float16).float()  # 8 significant bits, half up
    r = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    return torch.round(g * r[..., None]).clamp_(-7, 7), s


def _values(codes, s):
    return (codes * s[..., None]).flatten(-2)


def _nibbles(b):
    """[..., 4] bytes of words -> [..., 8] codes, lowest bits first."""
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _words(u):
    """[..., 8] codes -> [..., 4] bytes of words."""
    u = u.to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _unpack(pages, kv, d, page):
    """K and V as f32 [..., page, kv, d] of pages' bytes [..., page bytes]."""
    lead, groups = pages.shape[:-1], d // 32
    b = pages.reshape(*lead, kv, page * (d + d // 8))
    kc, vc, ks, vs = b.split([page * d // 2, page * d // 2, page * d // 16, page * d // 16], -1)
    k = _nibbles(kc.reshape(*lead, kv, page, 4, groups, 4)).transpose(-3, -2).reshape(*lead, kv, page, groups, 32)
    v = _nibbles(vc.reshape(*lead, kv, page // 8, d, 4)).transpose(-2, -1).reshape(*lead, kv, page, groups, 32)
    scale = lambda s: s.contiguous().view(torch.float16).reshape(*lead, kv, groups, page).transpose(-2, -1).float()  # noqa: E731
    back = lambda u, s: _values(u.float() - 8.0, scale(s)).movedim(-3, -2)  # noqa: E731
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


def _u32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _offsets(n):
    return _u32([0] + list(torch.tensor(n).cumsum(0).tolist()))


class State:
    """What a program holds before a call; `handle` is its cache object, made when first needed."""

    handle = None


def _pages_for(s, c, seed, lengths):
    """A pool in which the sequences' pages lie in any order, and the table that finds them."""
    g, page = _gen(seed + 1), c["page"]
    need = [-(-n // page) for n in lengths]
    s.max_pages = max(need) + 1
    s.pages = sum(need) + 3
    order = torch.randperm(s.pages, generator=g, device=DEV).to(torch.int32)
    s.table = torch.full((c["seqs"], s.max_pages), -1, dtype=torch.int32, device=DEV)
    first = 0
    for i, n in enumerate(need):
        s.table[i, :n] = order[first:first + n]
        first += n


def _fill(s, c, seed):
    g, page = _gen(seed + 2), c["page"]
    s.pool = torch.empty(s.pages, _page_bytes(c["kv"], c["d"], page), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (c["kv"] * page * c["d"]))
    for at in range(0, s.pages, step):  # a part at a time, so that the values fit
        n = min(step, s.pages - at)
        s.pool[at:at + n] = _pack(*(_randn(g, n, c["kv"], page, c["d"]) for _ in range(2)), c["kv"], c["d"], page)


def prepare(case, seed):
    c, s = case, State()
    s.c = c
    g = _gen(seed)
    if c["op"] == "append":
        n = _split(c)
        s.n, s.starts = n, [c["begin"] + 3 * i if c["begin"] else 0 for i in range(c["seqs"])]
        t = TYPES[c["type"]]
        s.q = _randn(g, c["rows"], c["heads"], c["d"]).to(t)
        s.k = _randn(g, c["rows"], c["kv"], c["d"]).to(t)
        s.v = _randn(g, c["rows"], c["kv"], c["d"]).to(t)
        s.offsets, s.begin = _offsets(n), _u32(s.starts)
        last = max(a + b for a, b in zip(s.starts, n))
        freq = 1e6 ** (-torch.arange(0, c["d"], 2, device=DEV, dtype=torch.float64) / c["d"])
        angle = torch.arange(last, device=DEV, dtype=torch.float64)[:, None] * freq
        s.rope = torch.stack([angle.cos(), angle.sin()], -1).float()  # [positions][d / 2] (cos, sin)
        _pages_for(s, c, seed, [a + b for a, b in zip(s.starts, n)])
        s.pool = torch.zeros(s.pages, _page_bytes(c["kv"], c["d"], c["page"]), dtype=torch.uint8, device=DEV)
        s.row_seq = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), torch.tensor(n, device=DEV))
    elif c["op"] == "read":
        n = _split(c)
        s.n, s.starts = n, [c["begin"] + 3 * i if c["begin"] else 0 for i in range(c["seqs"])]
        s.offsets, s.begin = _offsets(n), _u32(s.starts)
        _pages_for(s, c, seed, [a + b for a, b in zip(s.starts, n)])
        _fill(s, c, seed)
        s.row_seq = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), torch.tensor(n, device=DEV))
    elif c["op"] == "decode":
        s.n = _counts(c)
        s.lengths = _u32(s.n)
        _pages_for(s, c, seed, s.n)
        _fill(s, c, seed)
        s.q = _randn(g, c["seqs"], c["heads"], c["d"]).to(TYPES[c["type"]])
    elif c["op"] == "packed":
        s.n = _counts(c)
        s.nk = [x + c["before"] for x in s.n]
        s.q_offsets, s.k_offsets = _offsets(s.n), _offsets(s.nk)
        t = TYPES[c["type"]]
        s.q = _randn(g, sum(s.n), c["heads"], c["d"]).to(t)
        s.k = _randn(g, sum(s.nk), c["kv"], c["d"]).to(t)
        s.v = _randn(g, sum(s.nk), c["kv"], c["d"]).to(t)
    else:
        stride = c["layers"] * _page_bytes(c["kv"], c["d"], c["page"])
        s.pool = torch.randint(0, 256, (c["pages"], stride), dtype=torch.uint8, device=DEV, generator=g)
        order = torch.randperm(c["pages"], generator=g, device=DEV)[: 2 * c["count"]].to(torch.int32)
        s.pairs = order.reshape(2, c["count"]).t().contiguous()  # (from, to)
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------------------

_device = None


def _cache(s):
    """The program's device and the cache object over its pool."""
    global _device
    from enargeia_amd import kernels, kv4

    if _device is None:
        _device = kernels.Device(0)
    if s.handle is None:
        c = s.c
        s.handle = kv4.Kv4Cache(_device, kv_heads=c["kv"], head_dim=c["d"], page_size=c["page"], pages=s.pool.shape[0],
                                layers=c.get("layers", 1), pool=s.pool)
    return s.handle


def _run_own(s):
    c = s.c
    new = lambda *shape, t: torch.empty(*shape, dtype=TYPES[t], device=DEV)  # noqa: E731
    if c["op"] == "append":
        cache = _cache(s)
        q = new(c["rows"], c["heads"], c["d"], t=c["out"])
        k, v = (new(c["rows"], c["kv"], c["d"], t="f16") for _ in range(2))
        cache.append(s.k, s.v, s.offsets, s.begin, s.table, rows=c["rows"], sequences=c["seqs"], max_pages=s.max_pages,
                     q=s.q, q_out=q, heads=c["heads"], rope=s.rope, rope_positions=s.rope.shape[0],
                     in_type=c["type"], out_type=c["out"])
        cache.read(k, v, s.offsets, s.begin, s.table, rows=c["rows"], sequences=c["seqs"], max_pages=s.max_pages,
                   out_type="f16")
        return {"q": q, "k": k, "v": v}
    if c["op"] == "read":
        k, v = (new(c["rows"], c["kv"], c["d"], t=c["out"]) for _ in range(2))
        _cache(s).read(k, v, s.offsets, s.begin, s.table, rows=c["rows"], sequences=c["seqs"], max_pages=s.max_pages,
                       out_type=c["out"])
        return {"k": k, "v": v}
    if c["op"] == "decode":
        out = new(c["seqs"], c["heads"], c["d"], t=c["type"])
        _cache(s).attend(s.q, s.lengths, s.table, out, heads=c["heads"], sequences=c["seqs"], max_pages=s.max_pages,
                         type=c["type"])
        return out
    if c["op"] == "packed":
        global _device
        from enargeia_amd import kernels, kv4

        if _device is None:
            _device = kernels.Device(0)
        out = new(s.q.shape[0], c["heads"], c["d"], t=c["type"])
        kv4.attention_packed(_device, s.q, s.k, s.v, out, s.q_offsets, s.k_offsets, sequences=c["seqs"],
                             rows=s.q.shape[0], key_rows=s.k.shape[0], heads=c["heads"], kv_heads=c["kv"],
                             head_dim=c["d"], type=c["type"])
        return out
    _cache(s).copy_pages(s.pairs, c["count"])
    return s.pool


def _rotate(x, rope):
    """x [rows, heads, d] turned by its rows' (cos, sin) [rows, d / 2, 2]."""
    h = x.shape[-1] // 2
    a, b, co, si = x[..., :h], x[..., h:], rope[:, None, :, 0], rope[:, None, :, 1]
    return torch.cat([a * co - b * si, b * co + a * si], -1)


def _positions(s):
    i = torch.arange(s.row_seq.numel(), device=DEV)
    return s.begin.long()[s.row_seq] + i - s.offsets.long()[s.row_seq]


def _run_plain(s):
    c = s.c
    if c["op"] == "append":
        rope = s.rope[_positions(s)]
        q = _rotate(s.q.float(), rope).to(TYPES[c["out"]])
        k, v = (_values(*_quantise(x)).half() for x in (_rotate(s.k.float(), rope), s.v.float()))
        return {"q": q, "k": k, "v": v}
    if c["op"] == "read":
        at, page = _positions(s), c["page"]
        k, v = _unpack(s.pool, c["kv"], c["d"], page)
        p = s.table.long()[s.row_seq, at // page]
        return {"k": k[p, at % page].to(TYPES[c["out"]]), "v": v[p, at % page].to(TYPES[c["out"]])}
    if c["op"] == "decode":
        n, kv, d, page = c["seqs"], c["kv"], c["d"], c["page"]
        k, v = _unpack(s.pool[s.table.long().clamp(min=0)], kv, d, page)  # [seqs, pages, page, kv, d]
        k, v = (x.reshape(n, -1, kv, d).transpose(1, 2) for x in (k, v))
        q = s.q.float().reshape(n, kv, -1, d)
        w = q @ k.transpose(2, 3).contiguous() * (1.0 / math.sqrt(d))
        w = w.masked_fill(torch.arange(k.shape[2], device=DEV) >= s.lengths[:, None, None, None], -math.inf)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        return ((w @ v) / w.sum(-1, keepdim=True)).reshape(n, c["heads"], d).to(s.q.dtype)
    if c["op"] == "packed":
        # padded to the longest, all sequences at once
        kv, d = c["kv"], c["d"]
        rows = lambda o, most: (o[:-1, None] + torch.arange(most, device=DEV)).long()  # noqa: E731
        qi, ki = rows(s.q_offsets, max(s.n)), rows(s.k_offsets, max(s.nk))
        q = s.q.float()[qi.clamp(max=s.q.shape[0] - 1)].reshape(c["seqs"], max(s.n), kv, -1, d).permute(0, 2, 3, 1, 4)
        k, v = (x.float()[ki.clamp(max=x.shape[0] - 1)].permute(0, 2, 1, 3)[:, :, None] for x in (s.k, s.v))
        w = q @ k.transpose(3, 4).contiguous() * (1.0 / math.sqrt(d))
        nq, nk = (o.diff()[:, None, None] for o in (s.q_offsets, s.k_offsets))
        seen = torch.arange(max(s.nk), device=DEV) <= (nk - nq + torch.arange(max(s.n), device=DEV)[:, None])
        w = w.masked_fill_(~seen[:, None, None], -math.inf)
        w = w.sub_(w.amax(-1, keepdim=True)).exp_()
        o = ((w @ v) / w.sum(-1, keepdim=True)).permute(0, 3, 1, 2, 4).reshape(c["seqs"], max(s.n), c["heads"], d)
        return o[qi < s.q_offsets[1:, None]].to(s.q.dtype)
    s.pool[s.pairs[:, 1].long()] = s.pool[s.pairs[:, 0].long()]
    return s.pool


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "copy":
        return {"bytes": 2 * c["count"] * c["layers"] * _page_bytes(c["kv"], c["d"], c["page"]), "flops": 0}
    held = 2 * c["kv"] * (c["d"] // 2 + c["d"] // 16) if "kv" in c else 0  # of one position
    if c["op"] == "append":  # rows in, turned queries and pages out; the pages' rows read, their values out
        width, kvw = c["heads"] * c["d"], 2 * c["kv"] * c["d"]
        return {"bytes": c["rows"] * ((width + kvw) * SIZE[c["type"]] + width * SIZE[c["out"]] + 2 * held + kvw * 2 + 4 * c["d"]),
                "flops": 3 * c["rows"] * (width + kvw)}
    if c["op"] == "read":
        return {"bytes": c["rows"] * (held + 2 * c["kv"] * c["d"] * SIZE[c["out"]]), "flops": 2 * c["rows"] * c["kv"] * c["d"]}
    n = _counts(c)
    if c["op"] == "decode":
        return {"bytes": sum(n) * held + 2 * c["seqs"] * c["heads"] * c["d"] * SIZE[c["type"]],
                "flops": 4 * c["d"] * c["heads"] * sum(n)}
    pairs = sum(x * c["before"] + x * (x + 1) // 2 for x in n)
    return {"bytes": c["d"] * SIZE[c["type"]] * (2 * sum(n) * c["heads"] + 2 * (sum(n) + c["seqs"] * c["before"]) * c["kv"]),
            "flops": 4 * c["d"] * c["heads"] * pairs}


# ---- the definition in 64 bits, sequence by sequence -------------------------------------------


def _held64(x):
    """The values the cache holds for rows x [..., d]."""
    g = x.double().unflatten(-1, (-1, 32))
    s = (g.abs().amax(-1, keepdim=True) / 7.0).clamp(max=MOST_SCALE)
    bits = s.to(torch.float16).view(torch.int16).int()
    s = torch.div(bits + 4, 8, rounding_mode="floor").mul(8).to(torch.int16).view(torch.float16).double()
    return torch.where(s > 0, torch.round(g / s.clamp(min=1e-30)).clamp(-7, 7) * s, 0.0).flatten(-2)


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


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "append":
        outs = {"q": [], "k": [], "v": []}
        first = 0
        for n, start in zip(s.n, s.starts):
            rows = slice(first, first + n)
            z = torch.view_as_complex(s.rope[start:start + n].double().contiguous())[:, None]
            for name, x in (("q", s.q), ("k", s.k)):
                x = x[rows].double()
                t = torch.complex(x[..., : c["d"] // 2], x[..., c["d"] // 2:]) * z
                y = torch.cat([t.real, t.imag], -1)
                outs[name].append(y if name == "q" else _held64(y))
            outs["v"].append(_held64(s.v[rows]))
            first += n
        return {name: torch.cat(x) for name, x in outs.items()}
    if c["op"] == "read":
        got = [_row64(s, i, a + n) for i, (a, n) in enumerate(zip(s.starts, s.n))]
        return {name: torch.cat([x[j][a:] for x, a in zip(got, s.starts)]) for j, name in enumerate("kv")}
    if c["op"] == "decode":
        out = torch.empty(c["seqs"], c["heads"], c["d"], dtype=torch.float64, device=DEV)
        for i, n in enumerate(s.n):
            k, v = _row64(s, i, n)
            for h in range(c["heads"]):
                j = h // (c["heads"] // c["kv"])
                p = torch.softmax((k[:, j] @ s.q[i, h].double()) / math.sqrt(c["d"]), 0)
                out[i, h] = p @ v[:, j]
        return out
    if c["op"] == "packed":
        out = torch.empty(s.q.shape, dtype=torch.float64, device=DEV)
        q0 = k0 = 0
        for n, nk in zip(s.n, s.nk):
            hidden = torch.ones(n, nk, dtype=torch.bool, device=DEV).triu(nk - n + 1)
            for h in range(c["heads"]):
                j = h // (c["heads"] // c["kv"])
                w = s.q[q0:q0 + n, h].double() @ s.k[k0:k0 + nk, j].double().t().contiguous() / math.sqrt(c["d"])
                out[q0:q0 + n, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ s.v[k0:k0 + nk, j].double()
            q0, k0 = q0 + n, k0 + nk
        return out
    return None
