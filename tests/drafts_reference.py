"""The operators of a speculative step in numpy float64, written from their definitions
(include/enargeia_hip.h), for the tests of the kernels."""

import numpy as np

from kv4_reference import attend

NO_ROW = 0xFFFFFFFF


def frequencies(rotary, theta, scaling="none", factor=1.0, context=0.0, low=1.0, high=4.0):
    i = np.arange(rotary // 2)
    if scaling == "base":
        theta = theta * factor ** (rotary / (rotary - 2))
    f = theta ** (-2.0 * i / rotary)
    if scaling == "linear":
        return f / factor
    if scaling in ("turns", "log_turns"):
        t = context * f / (2 * np.pi)
        w = (t - low) / (high - low) if scaling == "turns" else np.log(t / low) / np.log(high / low)
        w = np.clip(w, 0.0, 1.0)
        return f * (w + (1 - w) / factor)
    return f


def rotate(x, cs, rotary, layout):
    """x [rows, heads, d] (f32) by cs [rows, rotary / 2, 2], each product rounded to f32."""
    y = np.array(x, np.float32)
    a, b = (slice(0, rotary // 2), slice(rotary // 2, rotary)) if layout == "half" else (slice(0, rotary, 2), slice(1, rotary, 2))
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    u, w = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


def parent_of(parents, i):
    """Row i's parent, or None: without parents the row before it."""
    p = i - 1 if parents is None else int(parents[i])
    return p if 0 <= p < i else None


def sees(parents, n):
    """[n, n]: whether row i sees row j (itself, or above it)."""
    m = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j is not None:
            m[i, j] = True
            j = parent_of(parents, j)
    return m


def tree_seen(parents, n, length, have):
    """[n, length]: the positions each row sees, of those that `have` a place."""
    seen = np.zeros((n, length), bool)
    if n <= length:
        seen[:, : length - n] = True
        seen[:, length - n:] = sees(parents, n)
        seen[:, ~have] = False
    return seen


def tree_attend(q, k, v, scale, parents, have):
    """q [n, heads, D] of the rows that lie last of k and v [length, kv, D]."""
    seen = tree_seen(parents, len(q), len(k), have)
    return np.stack([attend(q[i], k, v, scale, seen[i]) for i in range(len(q))]), seen


def verify(logits, tokens, parents, draft, accept, draw, temperature):
    """One sequence: (path, next)."""
    x = np.asarray(logits, np.float64)
    n, vocab = x.shape

    def best(r):
        ok = x[r] > -np.inf
        return int(np.flatnonzero(ok & (x[r] == x[r][ok].max()))[0]) if ok.any() else 0

    def probabilities(r):
        with np.errstate(all="ignore"):
            e = np.exp((x[r] - x[r].max()) / np.float64(temperature))
            return e / e.sum()

    path = [0]
    while True:
        at = path[-1]
        children = [r for r in range(n) if parent_of(parents, r) == at]
        if not temperature > 0:
            to = [r for r in children if int(tokens[r]) == best(at)]
            if not to:
                return path, best(at)
            path.append(to[0])
            continue
        p = probabilities(at)
        broken = not np.all(np.isfinite(p))
        left, rejected, to = 1.0, [], None
        for r in children:
            t = int(tokens[r])
            pt = p[t] if t < vocab else 0.0
            if draft is not None:
                q = float(draft[at, t]) if t < vocab else 0.0
                ok = float(accept[r]) * q < pt
            else:
                again = t in rejected
                ok = not again and float(accept[r]) * left < pt
                if not ok and not again:
                    left -= pt
            if ok and not broken:
                to = r
                break
            rejected.append(t)
        if to is not None:
            path.append(to)
            continue
        if broken:
            return path, best(at)
        mass = p.copy()
        if draft is not None and rejected:
            mass = np.maximum(p - np.asarray(draft[at], np.float64), 0.0)
        elif draft is None:
            mass[[t for t in rejected if t < vocab]] = 0.0
        run = np.cumsum(mass)
        if not run[-1] > 0:
            return path, best(at)
        over = np.flatnonzero(run > np.float64(draw) * run[-1])
        return path, int(over[0]) if len(over) else int(np.flatnonzero(mass > 0)[-1])


def verify_all(logits, tokens, offsets, parents, draft, accept, draws, temperatures, max_rows):
    """path [sequences, max_rows], counts, next of packed rows."""
    s = len(offsets) - 1
    path = np.full((s, max_rows), NO_ROW, np.uint32)
    counts, token = np.zeros(s, np.uint32), np.full(s, NO_ROW, np.uint32)
    for i in range(s):
        r = slice(int(offsets[i]), int(offsets[i + 1]))
        n = r.stop - r.start
        if n == 0 or n > max_rows:
            continue
        got, token[i] = verify(logits[r], tokens[r], None if parents is None else parents[r], None if draft is None else draft[r],
                               None if accept is None else accept[r], 0.0 if draws is None else draws[i],
                               0.0 if temperatures is None else temperatures[i])
        counts[i] = len(got)
        path[i, : len(got)] = got
    return path, counts, token


def keep(P, table, path, counts, ns, lengths, page):
    """The pages of P (kv4_reference.Pages, one layer) after the rows are kept, and the new lengths."""
    pages = len(P.pool)
    new = []
    for s, n in enumerate(ns):
        length = int(lengths[s])
        if n > path.shape[1] or n > length:
            new.append(length)
            continue
        base, c = length - n, min(int(counts[s]), n)
        new.append(base + c)
        where = lambda p: int(table[s][p // page]) if p // page < len(table[s]) else pages  # noqa: E731
        rows = {}
        for i in range(c):
            j = int(path[s][i])
            if j < n and where(base + j) < pages and where(base + i) < pages:
                rows[i] = [_raw(P, where(base + j), (base + j) % page, h) for h in range(P.kv)]
        for i, raw in rows.items():
            for h in range(P.kv):
                _put_raw(P, where(base + i), (base + i) % page, h, raw[h])
    return np.array(new, np.uint32)


def _raw(P, p, slot, h):
    kw, vw, ks, vs = P._streams(p, h)
    return kw[slot].copy(), (vw[slot // 8] >> np.uint32(4 * (slot % 8))) & np.uint32(15), ks.view(np.uint16)[:, slot].copy(), vs.view(np.uint16)[:, slot].copy()


def _put_raw(P, p, slot, h, raw):
    kw, vw, ks, vs = P._streams(p, h)
    kw[slot] = raw[0]
    sh = np.uint32(4 * (slot % 8))
    vw[slot // 8] = (vw[slot // 8] & ~(np.uint32(15) << sh)) | (raw[1] << sh)
    ks.view(np.uint16)[:, slot] = raw[2]
    vs.view(np.uint16)[:, slot] = raw[3]
