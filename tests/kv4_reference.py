"""The 4-bit cache's format and the operators over it in numpy float64, written from their
definitions (include/enargeia_hip.h), for the tests of the kernels."""

from fractions import Fraction

import numpy as np

NO_PAGE = 0xFFFFFFFF


def scale_of(top):
    """absmax (f32) of groups -> their f16 scales."""
    t = np.minimum(np.asarray(top, np.float32) * np.float32(1.0 / 7.0), np.float32(9344.0))
    bits = (t.astype(np.float16).view(np.uint16).astype(np.uint32) + 4) & 0xFFF8
    return np.where(np.isfinite(top), bits, 0x7E00).astype(np.uint16).view(np.float16)


def quantize(x):
    """Codes (0..15) and scales of rows x [..., D] (f32)."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        s = scale_of(np.abs(g).max(-1))  # (numpy's max passes NaN on)
        s32 = s.astype(np.float32)
        r = np.where(s32 > 0, np.float32(1) / s32, np.float32(0))
        c = np.clip(np.rint(g * r[..., None]), -7, 7)
        c = np.where(np.isfinite(s32)[..., None], c, 0)
    return (c + 8).astype(np.uint8).reshape(x.shape), s


def held(x):
    """The values that the cache holds for rows x [..., D], float64."""
    c, s = quantize(x)
    return ((c.astype(np.float64) - 8).reshape(*s.shape, 32) * s.astype(np.float64)[..., None]).reshape(x.shape)


def rotate(x, cs):
    """x [rows, heads, D] by cs [rows, D/2, 2], f32, each product rounded."""
    h = x.shape[-1] // 2
    a, b = x[..., :h].astype(np.float32), x[..., h:].astype(np.float32)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def _nearest(x, bits, least):
    """x (a Fraction) to `bits` significant bits, or to a multiple of 2^least where that is coarser: to
    nearest, ties to even."""
    if x == 0:
        return x
    e = abs(x).numerator.bit_length() - abs(x).denominator.bit_length()
    if abs(x) < Fraction(2) ** e:
        e -= 1
    step = Fraction(2) ** max(e + 1 - bits, least)
    return round(x / step) * step  # (round() of a Fraction takes ties to even)


def by_the_text(group):
    """Codes (0..15) and scale of 32 finite values by the header's words, in rational arithmetic."""
    x = [Fraction(float(v)) for v in group]
    f32 = lambda v: _nearest(v, 24, -149)  # noqa: E731
    t = min(f32(max(abs(v) for v in x) * f32(Fraction(1, 7))), Fraction(9344))
    t = _nearest(t, 11, -24)
    step = Fraction(1, 1 << 21)
    while t >= 256 * step:
        step *= 2
    s = (t / step + Fraction(1, 2)).__floor__() * step
    if s == 0:
        return [8] * len(x), 0.0
    r = f32(1 / s)
    return [max(-7, min(7, round(f32(v * r)))) + 8 for v in x], float(s)


def halfway(rng):
    """Groups of 32 values (f32) of every significand of a scale, with all the values halfway between two of
    its codes, and that scale's codes by an exact division."""
    significands = [(128 + i) / 128 for i in range(128)]
    groups, divided = [], []
    for i, m in enumerate(significands * 2):
        s = m * 2.0 ** int(rng.integers(-12, 12) if i >= 128 else 0)
        ties = np.array([c + 0.5 for c in range(-7, 7)] * 2 + [7.0, -7.0, 3.0, 0.0])
        groups.append(np.asarray(ties * s, np.float32))
        divided.append(np.rint(ties) + 8)
    return np.stack(groups), np.stack(divided).astype(np.uint8)


class Pages:
    """A pool's bytes, one layer, and its rows as the format places them."""

    def __init__(self, pages, kv, d, page, fill=0, stride=None):
        self.kv, self.d, self.page = kv, d, page
        self.bytes = kv * page * (d + d // 8)
        self.pool = np.full((pages, stride or self.bytes), fill, np.uint8)

    def _streams(self, p, h):
        b = self.pool[p, h * self.bytes // self.kv:(h + 1) * self.bytes // self.kv]
        n, d = self.page, self.d
        at = np.cumsum([0, n * d // 2, n * d // 2, n * d // 16, n * d // 16])
        k, v, ks, vs = (b[at[i]:at[i + 1]] for i in range(4))
        return (k.view(np.uint32).reshape(n, 4, d // 32), v.view(np.uint32).reshape(n // 8, d),
                ks.view(np.float16).reshape(d // 32, n), vs.view(np.float16).reshape(d // 32, n))

    def put(self, p, slot, h, k, v):
        """One row's K and V [D] (f32) into a slot."""
        kw, vw, ks, vs = self._streams(p, h)
        for x, words, scales, is_k in ((k, kw, ks, True), (v, vw, vs, False)):
            c, s = quantize(np.asarray(x, np.float32))
            scales[:, slot] = s
            for i in range(self.d):
                if is_k:
                    w, at, sh = words[slot, i % 32 // 8], i // 32, 4 * (i % 8)
                else:
                    w, at, sh = words[slot // 8], i, 4 * (slot % 8)
                w[at] = (int(w[at]) & ~(15 << sh) & 0xFFFFFFFF) | (int(c[i]) << sh)

    def get(self, p, slot, h):
        """One row's K and V, float64."""
        kw, vw, ks, vs = self._streams(p, h)
        i = np.arange(self.d)
        kc = (kw[slot, i % 32 // 8, i // 32] >> (4 * (i % 8)).astype(np.uint32)) & 15
        vc = (vw[slot // 8] >> np.uint32(4 * (slot % 8))) & 15
        return ((kc.astype(np.float64) - 8) * ks[i // 32, slot].astype(np.float64),
                (vc.astype(np.float64) - 8) * vs[i // 32, slot].astype(np.float64))

    def rows(self, table, length):
        """K and V [length, kv, D] of a sequence whose pages the table row names, and which exist."""
        k = np.zeros((length, self.kv, self.d))
        v = np.zeros((length, self.kv, self.d))
        have = np.zeros(length, bool)
        for j in range(length):
            p = int(table[j // self.page]) if j // self.page < len(table) else NO_PAGE
            if p < len(self.pool):
                have[j] = True
                for h in range(self.kv):
                    k[j, h], v[j, h] = self.get(p, j % self.page, h)
        return k, v, have


def random_pages(rng, pages, kv, d, page, spread=1.0):
    """A pool of quantized normal rows, and the values it holds [pages, page, kv, D] (K, V)."""
    P = Pages(pages, kv, d, page)
    k, v = (np.asarray(rng.standard_normal((pages, page, kv, d)) * spread, np.float32) for _ in range(2))
    for p in range(pages):
        for h in range(kv):
            kw, vw, ks, vs = P._streams(p, h)
            c, s = quantize(k[p, :, h])
            ks[:] = s.T
            n = c.reshape(page, d // 32, 4, 8).astype(np.uint32)
            kw[:] = np.bitwise_or.reduce(n << (4 * np.arange(8, dtype=np.uint32)), -1).transpose(0, 2, 1)
            c, s = quantize(v[p, :, h])
            vs[:] = s.T
            n = c.reshape(page // 8, 8, d).astype(np.uint32)
            vw[:] = np.bitwise_or.reduce(n << (4 * np.arange(8, dtype=np.uint32))[None, :, None], 1)
    return P, held(k), held(v)


def attend(q, k, v, scale, seen):
    """softmax(scale q K^T) V for q [heads, D], k and v [n, kv, D], over the positions in `seen`."""
    heads, d = q.shape
    out = np.zeros((heads, d))
    if not seen.any():
        return out
    group = heads // k.shape[1]
    for h in range(heads):
        w = scale * (k[seen, h // group] @ q[h].astype(np.float64))
        w = np.exp(w - w.max())
        out[h] = (w / w.sum()) @ v[seen, h // group]
    return out


def as_type(x, kind):
    """x as an element type: the array to upload, and its values in float64."""
    if kind == "bf16":
        b = np.ascontiguousarray(x, np.float32).view(np.uint32)
        b = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
        return b, (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    a = np.ascontiguousarray(x, np.float16 if kind == "f16" else np.float32)
    return a, a.astype(np.float64)


def from_type(raw, kind):
    """Raw bytes of an element type as float64."""
    if kind == "bf16":
        return (np.frombuffer(raw, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.frombuffer(raw, np.float16 if kind == "f16" else np.float32).astype(np.float64)


# Half a step of each type, relative: what one rounding may be off by.
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
