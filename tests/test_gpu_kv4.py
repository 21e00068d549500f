"""The operators over the paged 4-bit cache against their definitions in float64
(kv4_reference.py): append and read bit for bit, page copies byte for byte, the attentions within
bounds that count their roundings.

Bounds of an attention's output element. With A = sum_j p_j |V_j| (p normalised), an error e of every
score changes the weights by e^(2 e) - 1 at most, and each weight's own rounding w adds w A:
  scores: products of the queries' f16 parts (22 bits of the head's largest query for f32, exact for
    f16 and bf16) with exact codes, summed in f32 with the scale of each 32: (D / 32 + 40) 2^-24 +
    2^-21 for f32, of scale sum |q K| + 2^-22 of it at the head's largest query;
  weights: exp2 2^-22, its argument's rounding (|score| + 15) 2^-23, and their f16 parts: 2^-21 for f32
    rows, 2^-11 else, but no finer than half the last place of a denormal f16: weights are scaled so that the
    largest is 2^15, so 2^-25 / 2^15 = 2^-40 of the largest weight, which is at most their sum - with n
    of them n 2^-40 max |V| at most, all there is to go by where the large weights' values are 0;
  sums: one rounding per step of a lane, (positions / 32 + 24) 2^-24;
and the output's half step.
"""

import ctypes

import numpy as np
import pytest

from enargeia_amd import _lib, kv4
from enargeia_amd import kernels as K
from kv4_reference import (HALF_STEP, NO_PAGE, Pages, as_type, attend, from_type, held, random_pages, rotate)

pytestmark = pytest.mark.gpu


@pytest.fixture
def up(device):
    """Uploads that are released when the test ends."""
    held_buffers = []

    def make(a):
        b = device.upload(np.ascontiguousarray(a)) if isinstance(a, np.ndarray) else device.buffer(a)
        held_buffers.append(b)
        return b

    yield make
    device.sync()
    for b in held_buffers:
        b.release()


def tables(rng, lengths, page, pages, width):
    """A table whose sequences' pages lie in any order."""
    order = rng.permutation(pages)
    t = np.full((len(lengths), width), NO_PAGE, np.uint32)
    at = 0
    for i, n in enumerate(lengths):
        c = -(-n // page)
        t[i, :c] = order[at:at + c]
        at += c
    return t


def offsets_of(lengths, first=0):
    return np.concatenate([[first], first + np.cumsum(lengths)]).astype(np.uint32)


# ---- append and read ------------------------------------------------------------------------------


def check_append(device, up, rng, lengths, starts, heads, kv, d, page, in_type, out_type, before=0, after=0,
                 pad=0, rope=True, with_q=True):
    rows = before + sum(lengths) + after
    ends = [s + n for s, n in zip(starts, lengths)]
    width = max(-(-e // page) for e in ends) + 1
    pages = sum(-(-e // page) for e in ends) + 2
    table = tables(rng, ends, page, pages, width)
    P = Pages(pages, kv, d, page)
    P.pool[:] = rng.integers(0, 256, P.pool.shape, dtype=np.uint8)
    pool = up(P.pool.copy())
    strides = {"q": heads * d + pad, "k": kv * d + pad, "v": kv * d + 2 * pad}
    x = {n: rng.standard_normal((rows, s)).astype(np.float32) for n, s in strides.items()}
    raw = {n: as_type(a, in_type) for n, a in x.items()}
    vals = {n: np.asarray(raw[n][1], np.float32)[:, : (heads if n == "q" else kv) * d].reshape(rows, -1, d) for n in x}
    buf = {n: up(raw[n][0]) for n in x}
    angle = np.arange(max(ends) + 1)[:, None] * 1e4 ** (-np.arange(0, d, 2) / d)
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    mark = 0x5A
    outs = {n: up(np.full((rows, (heads if n == "q" else kv) * d * kv4_size(out_type)), mark, np.uint8)) for n in x}
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=pool)
    off = offsets_of(lengths, before)
    cache.append(buf["k"], buf["v"], up(off), up(np.array(starts, np.uint32)), up(table), rows=rows,
                 sequences=len(lengths), max_pages=width, q=buf["q"] if with_q else None,
                 q_out=outs["q"] if with_q else None, k_out=outs["k"], v_out=outs["v"], heads=heads if with_q else 0,
                 rope=up(cs) if rope else None, rope_positions=len(cs) if rope else 0, in_type=in_type,
                 out_type=out_type, q_stride=strides["q"] if pad else 0, k_stride=strides["k"] if pad else 0,
                 v_stride=strides["v"] if pad else 0)
    position = np.concatenate([np.arange(s, e) for s, e in zip(starts, ends)]).astype(int)
    seq = np.repeat(np.arange(len(lengths)), lengths)
    live = slice(before, before + sum(lengths))
    turned = {n: rotate(vals[n][live], cs[position]) if rope and n != "v" else vals[n][live] for n in x}
    for n in x if with_q else ("k", "v"):
        got = device.read(outs[n], rows * (heads if n == "q" else kv) * d * kv4_size(out_type))
        want = np.full((rows, (heads if n == "q" else kv) * d * kv4_size(out_type)), mark, np.uint8)
        want[live] = np.ascontiguousarray(as_type(turned[n].reshape(sum(lengths), -1), out_type)[0]).view(np.uint8)
        np.testing.assert_array_equal(np.frombuffer(got, np.uint8).reshape(want.shape), want, err_msg=f"{n} out")
    for i in range(sum(lengths)):
        p = table[seq[i], position[i] // page]
        for h in range(kv):
            P.put(p, position[i] % page, h, turned["k"][i, h], turned["v"][i, h])
    got = device.read_array(pool, np.uint8, P.pool.size).reshape(P.pool.shape)
    np.testing.assert_array_equal(got, P.pool, err_msg="pool")
    # read back what the rows' positions hold, in each type
    for t in ("f32", "f16", "bf16"):
        ko, vo = (up(np.full((rows, kv * d * kv4_size(t)), mark, np.uint8)) for _ in range(2))
        cache.read(ko, vo, up(off), up(np.array(starts, np.uint32)), up(table), rows=rows, sequences=len(lengths),
                   max_pages=width, out_type=t)
        for o, n in ((ko, "k"), (vo, "v")):
            want = np.full((rows, kv * d * kv4_size(t)), mark, np.uint8)
            want[live] = np.ascontiguousarray(as_type(held(turned[n]).reshape(sum(lengths), -1).astype(np.float32), t)[0]).view(np.uint8)
            got = device.read_array(o, np.uint8, want.size).reshape(want.shape)
            np.testing.assert_array_equal(got, want, err_msg=f"{n} read as {t}")


def kv4_size(kind):
    return 4 if kind == "f32" else 2


@pytest.mark.parametrize("lengths,starts", [
    ([1], [0]), ([1], [77]), ([3], [6]), ([8], [0]), ([9], [7]), ([1, 1, 1, 1, 1], [0, 7, 8, 31, 63]),
    ([40, 1, 0, 17, 100], [0, 5, 9, 33, 62]), ([0, 0, 5, 0], [1, 2, 3, 4])])
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 64), (4, 1, 128, 32)])
def test_append_and_read(device, up, lengths, starts, heads, kv, d, page):
    print(f"append {lengths} at {starts}, {heads}/{kv} x {d}, page {page}", flush=True)
    check_append(device, up, np.random.default_rng(len(lengths) + d), lengths, starts, heads, kv, d, page, "f32", "f16")


@pytest.mark.parametrize("in_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
def test_append_types(device, up, in_type, out_type):
    for d in (64, 128):
        check_append(device, up, np.random.default_rng(5), [70, 3], [5, 0], 3, 3, d, 128, in_type, out_type)


def test_append_packed_rows_outside_the_sequences_and_strides(device, up):
    rng = np.random.default_rng(6)
    check_append(device, up, rng, [5, 33], [2, 60], 6, 2, 64, 32, "f32", "f32", before=3, after=9, pad=4)
    check_append(device, up, rng, [11], [0], 8, 4, 128, 64, "f16", "bf16", before=70, after=1, pad=8, rope=False)
    check_append(device, up, rng, [11, 2], [0, 3], 8, 4, 64, 256, "bf16", "f16", with_q=False)


def test_append_long_rows_take_whole_blocks(device, up):
    # over 2048 rows a wave takes the blocks of 8 rows
    check_append(device, up, np.random.default_rng(7), [1500, 3, 800], [3, 8, 0], 2, 1, 64, 64, "f16", "f16", before=5)


def test_append_many_sequences(device, up):
    # more sequences than a wave reads offsets at a time, empty ones among them
    rng = np.random.default_rng(8)
    lengths = [int(n) for n in rng.integers(0, 4, 200)]
    check_append(device, up, rng, lengths, [int(s) for s in rng.integers(0, 40, 200)], 2, 1, 64, 32, "f32", "f16")


def test_values_at_the_edges(device, up):
    """Zeros, tiny and huge values, infinities and NaN: scales and codes as the format says."""
    d, page, n = 64, 32, 12
    x = np.random.default_rng(9).standard_normal((n, d)).astype(np.float32)
    for i, f in enumerate((0.0, 1e-30, 2.0 ** -20, 2.0 ** -18, 1e4, 65408.0, 1e30)):
        x[i] *= np.float32(f)
    x[7, 3], x[8, 40], x[9, 0], x[10, :32] = np.inf, np.nan, -np.inf, 7.0
    P = Pages(1, 1, d, page)
    pool = up(P.pool.copy())
    cache = kv4.Kv4Cache(device, 1, d, 1, page, pool=pool)
    b, off, st, tb = up(x), up(np.array([0, n], np.uint32)), up(np.zeros(1, np.uint32)), up(np.zeros(1, np.uint32))
    cache.append(b, b, off, st, tb, rows=n, sequences=1, max_pages=1)
    for i in range(n):
        P.put(0, i, 0, x[i], x[i])
    got = device.read_array(pool, np.uint8, P.pool.size).reshape(P.pool.shape)
    np.testing.assert_array_equal(got, P.pool)
    k, v = up(n * d * 4), up(n * d * 4)
    cache.read(k, v, off, st, tb, rows=n, sequences=1, max_pages=1, out_type="f32")
    for o in (k, v):
        np.testing.assert_array_equal(device.read_array(o, np.float32, n * d).reshape(n, d), held(x).astype(np.float32))


def test_rows_that_the_table_the_pages_or_the_rope_do_not_reach(device, up):
    """Such rows are skipped (append) or zeros (read), the others as ever."""
    rng = np.random.default_rng(10)
    d, page, n = 64, 32, 40
    x = rng.standard_normal((2 * n, d)).astype(np.float32)
    P = Pages(3, 1, d, page)
    P.pool[:] = rng.integers(0, 256, P.pool.shape, dtype=np.uint8)
    pool = up(P.pool.copy())
    # sequence 0: positions 20..59, its second page is none; sequence 1: 50..89 of a table of 64 positions
    table = np.array([[2, 3], [0, 1]], np.uint32)
    cs = np.tile(np.array([1.0, 0.0], np.float32), (62, d // 2, 1))  # the rope ends at 62
    b, out = up(x), up(np.full((2 * n, d), 9.0, np.float32))
    off, st, tb = up(np.array([0, n, 2 * n], np.uint32)), up(np.array([20, 50], np.uint32)), up(table)
    cache = kv4.Kv4Cache(device, 1, d, 3, page, pool=pool)
    cache.append(b, b, off, st, tb, rows=2 * n, sequences=2, max_pages=2, k_out=out, rope=up(cs), rope_positions=62)
    want = np.full((2 * n, d), 9.0, np.float32)
    want[:n] = x[:n]
    want[n:n + 12] = x[n:n + 12]
    np.testing.assert_array_equal(device.read_array(out, np.float32, want.size).reshape(want.shape), want)
    for i in range(12):
        P.put(2, 20 + i, 0, x[i], x[i])
        P.put(1, 50 + i - 32, 0, x[n + i], x[n + i])
    np.testing.assert_array_equal(device.read_array(pool, np.uint8, P.pool.size).reshape(P.pool.shape), P.pool)
    ko, vo = up(np.full((2 * n, d), 9.0, np.float32)), up(np.full((2 * n, d), 9.0, np.float32))
    cache.read(ko, vo, off, st, tb, rows=2 * n, sequences=2, max_pages=2, out_type="f32")
    got = device.read_array(ko, np.float32, want.size).reshape(want.shape)
    np.testing.assert_array_equal(got[:12], held(x[:12]))
    assert not got[12:n].any() and not got[n + 14:].any()
    np.testing.assert_array_equal(got[n:n + 12], held(x[n:n + 12]))


def test_starts_past_every_table(device, up):
    """Positions that no table reaches and whose sum with a row's index passes 32 bits: skipped, zeros."""
    rng = np.random.default_rng(40)
    d, page, n = 64, 32, 12
    x = rng.standard_normal((2 * n, d)).astype(np.float32)
    P = Pages(3, 1, d, page, fill=0x3C)
    pool = up(P.pool.copy())
    b, off, tb = up(x), up(np.array([0, n, 2 * n], np.uint32)), up(np.array([[2, 1], [0, 1]], np.uint32))
    st = up(np.array([0xFFFFFFFC, 0x7FFFFFFE], np.uint32))
    cs = up(np.ones((64, d // 2, 2), np.float32))
    ko, qo = (up(np.full((2 * n, d), 9.0, np.float32)) for _ in range(2))
    cache = kv4.Kv4Cache(device, 1, d, 3, page, pool=pool)
    for rope in (None, cs):
        cache.append(b, b, off, st, tb, rows=2 * n, sequences=2, max_pages=2, q=b, q_out=qo, heads=1, k_out=ko, rope=rope,
                     rope_positions=64)
        for o in (ko, qo):
            assert np.all(device.read_array(o, np.float32, x.size) == 9.0)
    np.testing.assert_array_equal(device.read_array(pool, np.uint8, P.pool.size).reshape(P.pool.shape), P.pool)
    cache.read(ko, qo, off, st, tb, rows=2 * n, sequences=2, max_pages=2, out_type="f32")
    for o in (ko, qo):
        assert not device.read_array(o, np.float32, x.size).any()


def test_offsets_that_do_not_ascend_end(device, up):
    """What they select is not said, but the calls end and keep to the rows and the sequences' pages."""
    d, page, n = 64, 32, 12
    b = up(np.ones((n, d), np.float32))
    off, st, tb = up(np.array([0, 5, 3, 10], np.uint32)), up(np.zeros(3, np.uint32)), up(np.array([[0], [1], [2]], np.uint32))
    P = Pages(4, 1, d, page, fill=0x3C)
    pool, out = up(P.pool.copy()), up(np.full((n, d), 9.0, np.float32))
    cache = kv4.Kv4Cache(device, 1, d, 4, page, pool=pool)
    cache.append(b, b, off, st, tb, rows=n, sequences=3, max_pages=1, q=b, q_out=out, heads=1, k_out=up(b.size))
    cache.read(out, up(b.size), off, st, tb, rows=n, sequences=3, max_pages=1, out_type="f32")
    kv4.attention_packed(device, b, b, b, up(b.size), off, off, sequences=3, rows=n, key_rows=n, heads=1, kv_heads=1,
                         head_dim=64)
    assert np.all(device.read_array(out, np.float32, n * d).reshape(n, d)[10:] == 9.0)
    assert np.all(device.read_array(pool, np.uint8, P.pool.size).reshape(P.pool.shape)[3] == 0x3C)


# ---- decode attention -------------------------------------------------------------------------------


def decode_bound(q, k, v, scale, seen, out, kind, out_kind=None):
    """The bound of the module's docstring, per head and dim."""
    heads, d = q.shape
    a = np.zeros((heads, d))
    n = int(seen.sum())
    if n == 0:
        return a
    for h in range(heads):
        kk, vv = k[seen, h // (heads // k.shape[1])], v[seen, h // (heads // k.shape[1])]
        s = scale * (kk @ q[h])
        w = np.exp(s - s.max())
        w /= w.sum()
        size = scale * (np.abs(kk) @ np.abs(q[h])).max()
        largest = scale * np.abs(kk).sum(-1).max() * np.abs(q[h]).max()
        e = size * (d / 32 + 40) * 2.0 ** -24 + (size * 2.0 ** -21 + largest * 2.0 ** -22 if kind == "f32" else 0.0)
        weight = 2.0 ** -22 + (np.abs(s).max() + 15) * 2.0 ** -23 + (2.0 ** -21 if kind == "f32" else 2.0 ** -11)
        a[h] = (w @ np.abs(vv)) * (np.expm1(2 * e) + weight + (n / 32 + 24) * 2.0 ** -24)
        a[h] += n * 2.0 ** -40 * np.abs(vv).max()
    return a + HALF_STEP[out_kind or kind] * np.abs(out) + 1e-30


def check_decode(device, up, rng, lengths, heads, kv, d, page, kind, extra=0, pad=0, scale=0.0, q_of=None, hole=None,
                 sequences=None):
    pages = sum(-(-n // page) for n in lengths) + 1
    width = max(-(-n // page) for n in lengths) + 1 + extra
    P, kv_k, kv_v = random_pages(rng, pages, kv, d, page)
    table = tables(rng, lengths, page, pages, width)
    # beyond each sequence's end its last page holds NaN scales and any codes
    for i, n in enumerate(lengths):
        if n % page:
            for h in range(kv):
                _, _, ks, vs = P._streams(table[i, n // page], h)
                ks[:, n % page:] = np.nan
                vs[:, n % page:] = np.inf
    if hole is not None:
        table[hole] = pages  # a page that is none
    q = rng.standard_normal((len(lengths), heads * d + pad)).astype(np.float32) if q_of is None else q_of
    raw, val = as_type(q, kind)
    out = up(np.full((len(lengths), (heads * d + pad) * kv4_size(kind)), 0x5A, np.uint8))
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(P.pool))
    cache.attend(up(raw), up(np.array(lengths, np.uint32)), up(table), out, heads=heads, sequences=len(lengths),
                 max_pages=width, type=kind, scale=scale, q_stride=heads * d + pad if pad else 0,
                 out_stride=heads * d + pad if pad else 0)
    got = from_type(device.read(out, q.size * kv4_size(kind)), kind).reshape(q.shape)
    tail = device.read_array(out, np.uint8, q.size * kv4_size(kind)).reshape(len(lengths), -1)[:, heads * d * kv4_size(kind):]
    assert np.all(tail == 0x5A)
    f = scale or 1.0 / np.sqrt(d)
    for i, n in enumerate(lengths):
        ids = table[i, : -(-n // page)]
        seen = (np.repeat(ids, page) < pages)[:n]
        ids = np.minimum(ids, pages - 1)
        k, v = (x[ids].reshape(-1, kv, d)[:n] for x in (kv_k, kv_v))
        qi = val[i, : heads * d].reshape(heads, d)
        want = attend(qi, k, v, f, seen)
        bound = decode_bound(qi, k, v, f, seen, want, kind)
        off = np.abs(got[i, : heads * d].reshape(heads, d) - want)
        assert np.all(off <= bound), (f"sequence {i} of {n}: off by {np.max(off / bound):.2f} of the bound", kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 64), (8, 8, 64, 32), (12, 4, 64, 256), (16, 1, 128, 128),
                                             (20, 1, 64, 64), (8, 1, 128, 64), (9, 3, 128, 32), (33, 1, 128, 256)])
def test_decode_lengths(device, up, heads, kv, d, page, kind):
    print(f"decode {heads}/{kv} x {d}, page {page}, {kind}", flush=True)
    rng = np.random.default_rng(heads + d + page)
    check_decode(device, up, rng, [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 700], heads, kv, d, page, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,extra", [([5000], 0), ([1], 900), ([513], 3000), ([3000, 0, 40, 1111], 10)])
def test_decode_splits(device, up, lengths, extra, kind):
    """A long axis split over workgroups and joined, and tables much wider than their sequences."""
    for heads, kv, d, page in ((14, 2, 64, 64), (16, 1, 128, 32)):
        print(f"decode {lengths} + {extra} pages, {heads}/{kv} x {d}, {kind}", flush=True)
        check_decode(device, up, np.random.default_rng(11), lengths, heads, kv, d, page, kind, extra=extra)


def test_decode_many_sequences(device, up):
    """More rows than the device holds at once, most of them of a position or none."""
    rng = np.random.default_rng(37)
    lengths = [int(n) for n in rng.integers(0, 3, 900)] + [100]
    check_decode(device, up, rng, lengths, 4, 2, 64, 64, "f32")
    check_decode(device, up, rng, lengths[600:], 3, 1, 128, 32, "f16")


def test_decode_tables_of_no_pages(device, up):
    """max_pages 0: no position is within reach, so nothing is attended to, stored or read."""
    P = Pages(1, 1, 64, 32)
    cache = kv4.Kv4Cache(device, 1, 64, 1, 32, pool=up(P.pool))
    x = np.ones((2, 64), np.float32)
    out, tb, two = up(np.full((2, 64), 7.0, np.float32)), up(np.zeros(2, np.uint32)), up(np.array([5, 9], np.uint32))
    cache.attend(up(x), two, tb, out, heads=1, sequences=2, max_pages=0)
    assert not device.read_array(out, np.float32, 128).any()
    off = up(np.array([0, 1, 2], np.uint32))
    cache.append(up(x), up(x), off, up(np.zeros(2, np.uint32)), tb, rows=2, sequences=2, max_pages=0)
    cache.read(out, out, off, up(np.zeros(2, np.uint32)), tb, rows=2, sequences=2, max_pages=0, out_type="f32")
    assert not device.read_array(out, np.float32, 128).any()
    assert not device.read_array(cache.pool, np.uint8, P.pool.size).any()


def test_decode_strides_scale_and_holes(device, up):
    rng = np.random.default_rng(12)
    check_decode(device, up, rng, [100, 300], 14, 2, 64, 64, "f32", pad=8, scale=0.3)
    check_decode(device, up, rng, [100, 300], 4, 2, 128, 32, "f16", pad=16, scale=0.01)
    check_decode(device, up, rng, [200, 300], 14, 2, 64, 64, "f32", hole=(1, 2))   # positions 128..191 of sequence 1
    check_decode(device, up, rng, [200, 600], 4, 2, 128, 32, "f32", hole=(0, slice(0, 7)))  # all of sequence 0: zeros


@pytest.mark.parametrize("factor", [0.0, 1e-30, 1e-4, 40.0, 3e3])
def test_decode_query_sizes(device, up, factor):
    """Scores from all equal to one that takes everything; heads of very different size side by side."""
    rng = np.random.default_rng(13)
    q = (rng.standard_normal((2, 14, 64)) * factor).astype(np.float32)
    q[:, ::2] *= np.float32(1e-3)
    check_decode(device, up, rng, [90, 500], 14, 2, 64, 64, "f32", q_of=q.reshape(2, -1))


def one_position_takes_all(s, v, got, half):
    """Rows of scores s [.., n] whose largest leads by far more than f32 rounds a score by: the result is its
    value, to the output's half step."""
    order = np.sort(s, -1)
    clear = order[..., -1] - order[..., -2] > 2.0 ** -18 * np.abs(s).max(-1) + 100.0
    assert clear.any()
    want = v[np.argmax(s, -1)]
    assert np.all(np.abs(got - want)[clear] <= (half + 2.0 ** -20) * np.abs(want)[clear])


@pytest.mark.parametrize("factor", [1e6, 1e9, 1e20])
def test_decode_scores_past_what_f32_resolves(device, up, factor):
    """Scores so large that a rounding of one is more than all exponents hold: still finite, the largest
    position's value."""
    rng = np.random.default_rng(35)
    heads, d, page, n = 4, 64, 64, 300
    P, k, v = random_pages(rng, 6, 1, d, page)
    table = rng.permutation(6)[None].astype(np.uint32)
    q = (rng.standard_normal((1, heads, d)) * factor).astype(np.float32)
    out = up(q.nbytes)
    cache = kv4.Kv4Cache(device, 1, d, 6, page, pool=up(P.pool))
    cache.attend(up(q), up(np.array([n], np.uint32)), up(table), out, heads=heads, sequences=1, max_pages=6)
    got = device.read_array(out, np.float32, q.size).reshape(heads, d)
    kk, vv = (x[table[0]].reshape(-1, d)[:n] for x in (k, v))
    assert np.isfinite(got).all()
    one_position_takes_all(q[0].astype(np.float64) @ kk.T / 8, vv, got, HALF_STEP["f32"])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [20, 32, 80, 200])
def test_decode_large_scores_where_half_a_step_has_no_position(device, up, n, d):
    """Steps of 64 positions of which a wave's first ends within the first 32."""
    rng = np.random.default_rng(37)
    heads, page = 4, 64
    P, k, v = random_pages(rng, 4, 1, d, page)
    table = rng.permutation(4)[None].astype(np.uint32)
    q = (rng.standard_normal((1, heads, d)) * 1e8).astype(np.float32)
    out = up(q.nbytes)
    cache = kv4.Kv4Cache(device, 1, d, 4, page, pool=up(P.pool))
    cache.attend(up(q), up(np.array([n], np.uint32)), up(table), out, heads=heads, sequences=1, max_pages=4)
    got = device.read_array(out, np.float32, q.size).reshape(heads, d)
    kk, vv = (x[table[0]].reshape(-1, d)[:n] for x in (k, v))
    assert np.isfinite(got).all()
    one_position_takes_all(q[0].astype(np.float64) @ kk.T / np.sqrt(d), vv, got, HALF_STEP["f32"])


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_decode_smallest_scale_and_queries(device, up, kind):
    """A scale and queries whose product is below f32: all positions alike, none past the end."""
    rng = np.random.default_rng(38)
    q = (rng.standard_normal((2, 4 * 64)) * 1e-35).astype(np.float32)
    check_decode(device, up, rng, [20, 300], 4, 1, 64, 64, kind, q_of=q, scale=1e-35)


def test_packed_smallest_scale(device, up):
    check_packed(device, up, np.random.default_rng(39), [70, 3], [70, 90], 2, 1, 64, "bf16", scale=1e-45)


@pytest.mark.parametrize("kind,factor", [("f16", 2e4), ("bf16", 1e6), ("bf16", 1e18)])
def test_packed_scores_past_what_f32_resolves(device, up, kind, factor):
    rng = np.random.default_rng(36)
    n, d = 200, 64

    def change(q, k, v):
        q *= np.float32(factor)
        if kind == "f16":
            q[:] = np.clip(q, -6e4, 6e4)
            k *= np.float32(1e4)

    (g, qi, ki, vi), = check_packed(device, up, rng, [1], [n], 2, 1, d, kind, change=change)
    assert np.isfinite(g).all()
    for h in range(2):
        # (its weight, not 1 where the running max lags, is rounded for the product and not for the sum: half a
        # step of it, and the output's)
        one_position_takes_all(qi[:, h] @ ki[:, 0].T / 8, vi[:, 0], g[:, h], 2 * HALF_STEP[kind])


def test_decode_not_finite_queries_and_rows_stay_where_they_are(device, up):
    rng = np.random.default_rng(14)
    heads, kv, d, page, n = 14, 2, 64, 64, 150
    P, k, v = random_pages(rng, 6, kv, d, page)
    table = np.array([[0, 1, 2], [3, 4, 5]], np.uint32)
    q = rng.standard_normal((2, heads, d)).astype(np.float32)
    q[0, 3, 5] = np.nan
    _, _, ks, vs = P._streams(4, 1)
    ks[0, 7] = np.nan  # sequence 1, kv head 1, position 71
    out = up(q.nbytes)
    cache = kv4.Kv4Cache(device, kv, d, 6, page, pool=up(P.pool))
    cache.attend(up(q), up(np.array([n, n], np.uint32)), up(table), out, heads=heads, sequences=2, max_pages=3)
    got = device.read_array(out, np.float32, q.size).reshape(q.shape)
    bad = np.zeros((2, heads), bool)
    bad[0, 3] = bad[1, 7:] = True
    np.testing.assert_array_equal(np.isnan(got).all(-1), bad)
    np.testing.assert_array_equal(np.isnan(got).any(-1), bad)
    cache.attend(up(q), up(np.array([n, 71], np.uint32)), up(table), out, heads=heads, sequences=2, max_pages=3)
    got = device.read_array(out, np.float32, q.size).reshape(q.shape)
    bad[1] = False  # the row is past the length
    np.testing.assert_array_equal(np.isnan(got).any(-1), bad)


def test_decode_length_past_the_table(device, up):
    """A length past the table's reach counts as its reach."""
    rng = np.random.default_rng(15)
    P, k, v = random_pages(rng, 2, 1, 64, 32)
    q = rng.standard_normal((1, 4, 64)).astype(np.float32)
    out = up(q.nbytes)
    cache = kv4.Kv4Cache(device, 1, 64, 2, 32, pool=up(P.pool))
    cache.attend(up(q), up(np.array([0xFFFFFFFF], np.uint32)), up(np.array([[1, 0]], np.uint32)), out, heads=4,
                 sequences=1, max_pages=2)
    got = device.read_array(out, np.float32, q.size).reshape(4, 64)
    kk, vv = (x[[1, 0]].reshape(-1, 1, 64) for x in (k, v))
    seen = np.ones(64, bool)
    want = attend(q[0], kk, vv, 0.125, seen)
    assert np.all(np.abs(got - want) <= decode_bound(q[0].astype(np.float64), kk, vv, 0.125, seen, want, "f32"))


def test_pool_past_4_gib(device, up):
    """Pages 128 MiB apart: append, read, attention and a copy at byte offsets past 32 bits."""
    rng = np.random.default_rng(16)
    kv, d, page, stride, pages = 1, 64, 32, 1 << 27, 36
    need = stride * (pages - 1) + kv4.page_bytes(kv, d, page)
    pool = up(need)
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=pool)
    cache.dims.page_stride = stride
    x = rng.standard_normal((2, 50, d)).astype(np.float32)
    table = np.array([[34, 33]], np.uint32)
    off, st, tb = up(np.array([0, 50], np.uint32)), up(np.zeros(1, np.uint32)), up(table)
    cache.append(up(x[0]), up(x[1]), off, st, tb, rows=50, sequences=1, max_pages=2)
    ko, vo = up(x[0].nbytes), up(x[0].nbytes)
    cache.read(ko, vo, off, st, tb, rows=50, sequences=1, max_pages=2, out_type="f32")
    np.testing.assert_array_equal(device.read_array(ko, np.float32, x[0].size).reshape(50, d), held(x[0]))
    np.testing.assert_array_equal(device.read_array(vo, np.float32, x[0].size).reshape(50, d), held(x[1]))
    cache.copy_pages(up(np.array([[34, 32], [33, 1]], np.uint32)), 2)
    q = rng.standard_normal((1, 3, d)).astype(np.float32)
    k, v = held(x[0])[:, None], held(x[1])[:, None]
    seen = np.ones(50, bool)
    want = attend(q[0], k, v, 0.125, seen)
    for t in (table, np.array([[32, 1]], np.uint32)):
        out = up(q.nbytes)
        cache.attend(up(q), up(np.array([50], np.uint32)), up(t), out, heads=3, sequences=1, max_pages=2)
        got = device.read_array(out, np.float32, q.size).reshape(3, d)
        assert np.all(np.abs(got - want) <= decode_bound(q[0].astype(np.float64), k, v, 0.125, seen, want, "f32"))


# ---- page copies ------------------------------------------------------------------------------------


@pytest.mark.parametrize("kv,d,page,layers,count", [(2, 64, 64, 24, 5), (1, 64, 32, 1, 1), (3, 128, 32, 3, 9)])
def test_copy_pages(device, up, kv, d, page, layers, count):
    rng = np.random.default_rng(17)
    pages = 2 * count + 3
    size = kv4.page_bytes(kv, d, page) * layers
    host = rng.integers(0, 256, (pages, size), dtype=np.uint8)
    pool = up(host)
    order = rng.permutation(pages)[: 2 * count].reshape(count, 2).astype(np.uint32)
    pairs = np.concatenate([order, np.array([[pages, 0], [0, 0xFFFFFFFF]], np.uint32)])  # two that are no pages
    kv4.Kv4Cache(device, kv, d, pages, page, layers=layers, pool=pool).copy_pages(up(pairs), count + 2)
    host[order[:, 1]] = host[order[:, 0]]
    np.testing.assert_array_equal(device.read_array(pool, np.uint8, host.size).reshape(host.shape), host)


# ---- packed attention -------------------------------------------------------------------------------


def packed_reference(q, k, v, nq, nk, scale, kind, out_kind):
    """Output and bound of one sequence: q [nq, heads, d], k, v [nk, kv, d]."""
    heads, d = q.shape[1:]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(heads):
        kk, vv = k[:, h // (heads // k.shape[1])], v[:, h // (heads // k.shape[1])]
        s = scale * (q[:, h] @ kk.T)
        see = np.arange(nk)[None] <= nk - nq + np.arange(nq)[:, None]
        rows = see.any(1)
        if not rows.any():
            continue
        s = np.where(see, s, -np.inf)[rows]
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[rows, h] = w @ vv
        size = scale * (np.abs(q[rows, h]) @ np.abs(kk).T).max(1, keepdims=True)
        # scores: f32 sums of D exact products; weights: exp2, its argument, and their own half step
        # (f16 weights under 2^-14 half a denormal step); sums: a rounding per 8 keys and tile
        e = size * (d + 4) * 2.0 ** -24
        weight = 2.0 ** -22 + (2 * size + 2) * 2.0 ** -23 + HALF_STEP[kind]
        flat = nk * 2.0 ** -25 * np.abs(vv).max(initial=0) if kind == "f16" else 0.0
        bound[rows, h] = (w @ np.abs(vv)) * (np.expm1(2 * e) + weight + (nk / 8 + 24) * 2.0 ** -24) + flat
    return out, bound + HALF_STEP[out_kind] * np.abs(out) + 1e-30


def check_packed(device, up, rng, nq, nk, heads, kv, d, kind, out_kind=None, before=0, after=0, pad=0, scale=0.0,
                 change=None):
    out_kind = out_kind or kind
    qo, ko = offsets_of(nq, before), offsets_of(nk, 2 * before)
    rows, key_rows = before + sum(nq) + after, 2 * before + sum(nk) + after
    strides = (heads * d + pad, kv * d + 2 * pad, kv * d + pad, heads * d + 3 * pad)
    q, k, v = (rng.standard_normal((r, s)).astype(np.float32) for r, s in zip((rows, key_rows, key_rows), strides))
    # rows of no sequence
    for x, o in ((q, qo), (k, ko), (v, ko)):
        x[: o[0]] = x[o[-1]:] = np.nan
    if change:
        change(q, k, v)
    (q, qv), (k, kx), (v, vx) = (as_type(x, kind) for x in (q, k, v))
    out = up(np.full((rows, strides[3] * kv4_size(out_kind)), 0x5A, np.uint8))
    kv4.attention_packed(device, up(q), up(k), up(v), out, up(qo), up(ko), sequences=len(nq), rows=rows,
                         key_rows=key_rows, heads=heads, kv_heads=kv, head_dim=d, type=kind, out_type=out_kind,
                         scale=scale, q_stride=strides[0] if pad else 0, k_stride=strides[1] if pad else 0,
                         v_stride=strides[2] if pad else 0, out_stride=strides[3] if pad else 0)
    raw = device.read_array(out, np.uint8, rows * strides[3] * kv4_size(out_kind)).reshape(rows, -1)
    live = raw[qo[0]:qo[-1], : heads * d * kv4_size(out_kind)]
    got = from_type(np.ascontiguousarray(live).tobytes(), out_kind).reshape(-1, heads, d)
    rest = raw.copy()
    rest[qo[0]:qo[-1], : heads * d * kv4_size(out_kind)] = 0x5A
    assert np.all(rest == 0x5A), "rows or columns outside the sequences were written"
    values = []
    for i in range(len(nq)):
        qi = qv[qo[i]:qo[i + 1], : heads * d].reshape(-1, heads, d)
        ki, vi = (x[ko[i]:ko[i + 1], : kv * d].reshape(-1, kv, d) for x in (kx, vx))
        values.append((got[qo[i] - qo[0]:qo[i + 1] - qo[0]], qi, ki, vi))
    if change:
        return values
    for i, (g, qi, ki, vi) in enumerate(values):
        want, bound = packed_reference(qi, ki, vi, nq[i], nk[i], scale or 1.0 / np.sqrt(d), kind, out_kind)
        off = np.abs(g - want)
        assert np.all(off <= bound), f"sequence {i}: off by {np.max(off / bound):.2f} of the bound"
    return None


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d", [(14, 2, 64), (2, 2, 64), (8, 2, 128), (3, 1, 128)])
@pytest.mark.parametrize("nq", [[1], [63], [64], [65], [129], [1, 0, 200, 7, 128, 31, 32, 33], [700]])
def test_packed_prompts(device, up, nq, heads, kv, d, kind):
    print(f"packed {nq}, {heads}/{kv} x {d}, {kind}", flush=True)
    check_packed(device, up, np.random.default_rng(sum(nq) + d), nq, nq, heads, kv, d, kind)


@pytest.mark.parametrize("heads,kv", [(14, 2), (16, 16), (24, 3), (20, 5), (12, 1), (16, 4)])
@pytest.mark.parametrize("sequences", [24, 70])
def test_packed_more_workgroups_than_cus(device, up, sequences, heads, kv):
    """Every query block is some workgroup's, however heads and blocks are laid over the XCDs."""
    rng = np.random.default_rng(41)
    nq = [int(n) for n in rng.integers(1, 60, sequences)]
    nq[3], nq[5] = 300, 0
    check_packed(device, up, rng, nq, nq, heads, kv, 64, "f16")


@pytest.mark.parametrize("nq,nk", [([5], [300]), ([64, 1], [65, 1000]), ([200, 130], [330, 128]), ([3, 4], [0, 2]),
                                   ([300], [40])])
def test_packed_chunks_after_earlier_rows_and_rows_that_see_nothing(device, up, nq, nk):
    for d, kind in ((64, "f16"), (128, "bf16")):
        check_packed(device, up, np.random.default_rng(21), nq, nk, 4, 2, d, kind)


@pytest.mark.parametrize("kind,out_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
def test_packed_few_queries_over_long_keys(device, up, kind, out_kind):
    """The keys split over workgroups and joined: sequences of very different lengths, some shorter than a
    split, blocks whose last splits are empty, queries that see nothing."""
    rng = np.random.default_rng(27)
    for heads, kv, d in ((3, 1, 64), (4, 4, 128), (6, 3, 64)):
        print(f"packed few queries, {heads}/{kv} x {d}, {kind} {out_kind}", flush=True)
        check_packed(device, up, rng, [130, 3, 1], [5000, 1100, 40], heads, kv, d, kind, out_kind, before=2, after=1)
        check_packed(device, up, rng, [200, 0, 70], [100, 9, 4200], heads, kv, d, kind, out_kind)
        check_packed(device, up, rng, [2500], [2500], heads, kv, d, kind, out_kind)


def test_packed_strides_types_and_rows_outside(device, up):
    rng = np.random.default_rng(22)
    check_packed(device, up, rng, [40, 90], [40, 90], 14, 2, 64, "f16", "f32", before=3, after=5, pad=8)
    check_packed(device, up, rng, [40, 90], [140, 90], 4, 1, 128, "bf16", "f32", before=1, after=70, pad=16, scale=0.2)
    check_packed(device, up, rng, [1] * 150 + [3], [2] * 150 + [70], 2, 1, 64, "f16", after=2)


@pytest.mark.parametrize("factor", [0.0, 1e-4, 30.0, 200.0])
def test_packed_query_sizes(device, up, factor):
    rng = np.random.default_rng(23)
    q = rng.standard_normal((150, 128)).astype(np.float32) * factor

    def change(a, k, v):
        a[:] = q

    for g, qi, ki, vi in check_packed(device, up, rng, [150], [150], 2, 1, 64, "bf16", change=change):
        want, bound = packed_reference(qi, ki, vi, 150, 150, 0.125, "bf16", "bf16")
        assert np.all(np.abs(g - want) <= bound)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("what", ["k", "v", "q"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_packed_not_finite_values_stay_with_who_sees_them(device, up, what, value, kind):
    """A key or value that is not finite reaches the queries from its position on, and no other."""
    n, at = 150, 70

    def change(q, k, v):
        x = {"q": q, "k": k, "v": v}[what]
        x[at, 5] = value

    (g, qi, ki, vi), = check_packed(device, up, np.random.default_rng(24), [n], [n], 2, 1, 64, kind, change=change)
    clean = {"q": qi, "k": ki, "v": vi}
    clean[what] = np.where(np.isfinite(clean[what]), clean[what], 0.0)
    want, bound = packed_reference(clean["q"], clean["k"], clean["v"], n, n, 0.125, kind, kind)
    if what == "q":
        assert np.isnan(g[at, 0]).all()
        ok = np.ones((n, 2), bool)
        ok[at, 0] = False
        assert np.all(np.abs(g - want)[ok] <= bound[ok])
    elif what == "k":
        assert np.all(np.abs(g - want)[:at] <= bound[:at])
        if np.isnan(value):
            assert np.isnan(g[at:]).all()
    else:
        assert not np.isfinite(g[at:, :, 5]).any()
        g, want, bound = (np.delete(x, 5, 2) if x is not None else x for x in (g, want, bound))
        assert np.all(np.abs(g - want) <= bound)
    if what == "v":
        return
    assert np.isfinite(g[:at]).all()


@pytest.mark.parametrize("nq,nk", [(150, 150), (150, 4000)])
def test_packed_value_before_the_poisoned_row_is_clean(device, up, nq, nk):
    at = nk - nq  # the first query's own position

    def change(q, k, v):
        v[at + 70, 5] = np.nan
        v[at + 100, 6] = np.inf

    (g, qi, ki, vi), = check_packed(device, up, np.random.default_rng(25), [nq], [nk], 2, 1, 128, "bf16", change=change)
    assert np.isfinite(g[:70]).all() and np.isnan(g[70:, :, 5]).all()
    assert np.isfinite(g[:100, :, 6]).all() and not np.isfinite(g[100:, :, 6]).any()


def test_packed_keys_past_4_gib(device, up):
    """Key rows 16 MiB apart: byte offsets past 32 bits."""
    rng = np.random.default_rng(26)
    n, stride, d = 300, 1 << 23, 64
    big = up(((n - 1) * stride + d) * 2)
    q, k = (rng.standard_normal((n, d)).astype(np.float16) for _ in range(2))
    for i in range(n):
        device.write(big, k[i], offset=i * stride * 2)
    device.sync()
    out, off = up(q.nbytes), up(np.array([0, n], np.uint32))
    kv4.attention_packed(device, up(q), big, big, out, off, off, sequences=1, rows=n, key_rows=n, heads=1, kv_heads=1,
                         head_dim=d, k_stride=stride, v_stride=stride)
    got = device.read_array(out, np.float16, q.size).reshape(n, 1, d).astype(np.float64)
    want, bound = packed_reference(q[:, None].astype(np.float64), *(k[:, None].astype(np.float64),) * 2, n, n, 0.125, "f16", "f16")
    assert np.all(np.abs(got - want) <= bound)


# ---- refusals -----------------------------------------------------------------------------------------


def test_refusals(device, up):
    b = up(1 << 16)
    cache = kv4.Kv4Cache(device, 2, 64, 3, 64, pool=b)
    ok = dict(rows=1, sequences=1, max_pages=1)

    def fails(match, call, error=_lib.EgError):
        with pytest.raises(error, match=match):
            call()

    def with_dims(match, error=_lib.EgError, **change):
        old = {n: getattr(cache.dims, n) for n in change}
        for n, x in change.items():
            setattr(cache.dims, n, x)
        for call in (lambda: cache.append(b, b, b, b, b, **ok), lambda: cache.read(b, b, b, b, b, **ok),
                     lambda: cache.attend(b, b, b, b, heads=2, sequences=1, max_pages=1)):
            fails(match, call, error)
        for n, x in old.items():
            setattr(cache.dims, n, x)

    with_dims("head_dim 96 is not supported", head_dim=96)
    with_dims("page_size 48 is not supported", page_size=48)
    with_dims("0 kv heads", kv_heads=0)
    with_dims("a pool of no pages", pages=0)
    with_dims("page_stride 9215 is not a multiple of 16 of at least 9216", page_stride=9215)
    with_dims("page_stride 9200 is not", page_stride=9200)
    fails("positions", lambda: cache.attend(b, b, b, b, heads=2, sequences=1, max_pages=1 << 26), _lib.EgRangeError)
    fails("2097152 sequences", lambda: cache.attend(b, b, b, b, heads=2, sequences=1 << 21, max_pages=1), _lib.EgRangeError)
    fails("heads 3 are not a multiple", lambda: cache.attend(b, b, b, b, heads=3, sequences=1, max_pages=1))
    fails("scale -1", lambda: cache.attend(b, b, b, b, heads=2, sequences=1, max_pages=1, scale=-1.0))
    fails("scale nan", lambda: cache.attend(b, b, b, b, heads=2, sequences=1, max_pages=1, scale=float("nan")))
    fails("strides 132", lambda: cache.attend(b, b, b, b, heads=2, sequences=1, max_pages=1, q_stride=132))
    fails("q and out must be 16-byte aligned", lambda: cache.attend(K.Binding(b, 4), b, b, b, heads=2, sequences=1, max_pages=1))
    fails("NULL argument", lambda: cache.attend(b, None, b, b, heads=2, sequences=1, max_pages=1))
    fails("q, q_out and heads go together", lambda: cache.append(b, b, b, b, b, q=b, heads=2, **ok))
    fails("q, q_out and heads go together", lambda: cache.append(b, b, b, b, b, q=b, q_out=b, **ok))
    fails("row strides", lambda: cache.append(b, b, b, b, b, k_stride=64, **ok))
    fails("row strides", lambda: cache.append(b, b, b, b, b, k_stride=130, **ok))
    fails("16-byte aligned", lambda: cache.append(K.Binding(b, 8), b, b, b, b, **ok))
    fails("element type 'q4'", lambda: cache.append(b, b, b, b, b, in_type="q4", **ok))
    fails("NULL argument", lambda: cache.read(b, None, b, b, b, **ok))
    fails("layer 1 of 1", lambda: cache.read(b, b, b, b, b, layer=1, **ok), _lib.EgRangeError)
    fails("NULL argument", lambda: cache.copy_pages(None, 1))
    fails("rows over the grid limit", lambda: cache.read(b, b, b, b, b, rows=1 << 29, sequences=1, max_pages=1),
          _lib.EgRangeError)
    cache.dims.page_stride = 1 << 50  # (times the count, past 64 bits)
    fails("over the grid limit", lambda: cache.copy_pages(b, 1 << 27), _lib.EgRangeError)
    cache.dims.page_stride = kv4.page_bytes(2, 64, 64)
    pk = dict(sequences=1, rows=1, key_rows=1, heads=2, kv_heads=1, head_dim=64)
    call = lambda **change: kv4.attention_packed(device, b, b, b, b, b, b, **{**pk, **change})  # noqa: E731
    fails("head_dim 80 is not supported", lambda: call(head_dim=80))
    fails("not a multiple of kv_heads", lambda: call(kv_heads=3))
    fails("type 0", lambda: call(type="f32"))
    fails("out_type 2", lambda: call(type="f16", out_type="bf16"))
    fails("strides 128, 60", lambda: call(k_stride=60))
    fails("strides", lambda: call(v_stride=68))
    fails("key strides", lambda: call(k_stride=1 << 24), _lib.EgRangeError)
    fails("1073741824 key rows", lambda: call(key_rows=1 << 30), _lib.EgRangeError)
    fails("scale inf", lambda: call(scale=float("inf")))
    # nothing to do is no error
    call(rows=0)
    call(sequences=0)
    cache.append(b, b, b, b, b, rows=0, sequences=1, max_pages=1)
    cache.attend(b, b, b, b, heads=2, sequences=0, max_pages=0)
    cache.copy_pages(None, 0)
    # nor are the pointers of arrays without an element
    kv4.attention_packed(device, None, None, None, None, b, b, **{**pk, "rows": 0})
    cache.append(None, None, b, b, b, heads=2, rows=0, sequences=1, max_pages=1)
    cache.read(None, None, None, None, None, rows=0, sequences=0, max_pages=0)
    cache.attend(None, None, None, None, heads=2, sequences=0, max_pages=0)
    fails("NULL argument", lambda: kv4.attention_packed(device, b, None, None, b, b, b, **pk))
    zeros, one = up(np.zeros(2, np.uint32)), up(np.array([0, 1], np.uint32))
    out = up(np.full((2, 128), 9.0, np.float16))
    kv4.attention_packed(device, b, None, None, out, one, zeros, **{**pk, "key_rows": 0})
    cache.attend(b, zeros, None, K.Binding(out, 256), heads=2, sequences=1, max_pages=0, type="f16")
    assert not device.read_array(out, np.float16, 256).any()
    device.sync()


# ---- together, captured, on other streams ----------------------------------------------------------


def serve(device, up, rng, capture):
    """Two prompts, a second chunk of one, a fork, decode steps of all - append, packed attention, read,
    page copies and decode attention as a program runs them - against float64 over the same values."""
    heads, kv, d, page, layers = 6, 2, 64, 32, 2
    layer = 1
    pages = kv4.PageTable(16, page)
    cache = kv4.Kv4Cache(device, kv, d, 16, page, layers=layers)
    angle = np.arange(256)[:, None] * 1e4 ** (-np.arange(0, d, 2) / d)
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    rope = up(cs)
    rows_of = {}  # what each sequence holds: K, V rows in float64
    scale = 1.0 / np.sqrt(d)

    def rows(n, h):
        return rng.standard_normal((n, h, d)).astype(np.float32)

    def chunk(seqs, lengths, whole):
        starts = [pages.grow(s, n) for s, n in zip(seqs, lengths)]
        copies = pages.take_copies()
        if len(copies):
            cache.copy_pages(up(copies), len(copies))
        n, table = sum(lengths), pages.table(seqs, 8)
        q, k, v = rows(n, heads), rows(n, kv), rows(n, kv)
        qo, ko, vo = up(q.nbytes // 2), up(k.nbytes // 2), up(k.nbytes // 2)
        off, st, tb = up(offsets_of(lengths)), up(np.array(starts, np.uint32)), up(table)
        common = dict(sequences=len(seqs), max_pages=8, layer=layer)
        cache.append(up(k), up(v), off, st, tb, rows=n, q=up(q), q_out=qo, k_out=ko, v_out=vo, heads=heads, rope=rope,
                     rope_positions=256, out_type="f16", **common)
        keys = [s + m for s, m in zip(starts, lengths)]
        koff, total = off, n
        if not whole:  # earlier rows too, as the cache holds them
            koff, total = up(offsets_of(keys)), sum(keys)
            ko, vo = up(total * kv * d * 2), up(total * kv * d * 2)
            cache.read(ko, vo, koff, up(np.zeros(len(seqs), np.uint32)), tb, rows=total, **common)
        out = up(q.nbytes)
        kv4.attention_packed(device, qo, ko, vo, out, off, koff, sequences=len(seqs), rows=n, key_rows=total,
                             heads=heads, kv_heads=kv, head_dim=d, out_type="f32")
        got = device.read_array(out, np.float32, q.size).reshape(q.shape)
        at = 0
        for s, m, b in zip(seqs, lengths, starts):
            r = slice(at, at + m)
            kr = rotate(k[r], cs[b:b + m])
            old = rows_of.get(s, (np.zeros((0, kv, d)), np.zeros((0, kv, d))))
            rows_of[s] = tuple(np.concatenate([x, held(y)]) for x, y in zip(old, (kr, v[r])))
            qr = rotate(q[r], cs[b:b + m]).astype(np.float16).astype(np.float64)
            kk, vv = (kr.astype(np.float16), v[r].astype(np.float16)) if whole else rows_of[s]
            want, bound = packed_reference(qr, kk.astype(np.float64), vv.astype(np.float64), m, b + m, scale, "f16", "f32")
            assert np.all(np.abs(got[r] - want) <= bound)
            at += m

    a, b = pages.create(), pages.create()
    chunk([a, b], [45, 70], True)
    chunk([b, a], [9, 30], False)
    c = pages.fork(b)
    rows_of[c] = rows_of[b]
    seqs = [c, a, b]
    q, k, v = (up(4 * 3 * h * d) for h in (heads, kv, kv))
    qo, out, off = up(4 * 3 * heads * d), up(4 * 3 * heads * d), up(offsets_of([1, 1, 1]))
    st, ln, tb = up(16), up(16), up(4 * 3 * 8)

    def launches():
        cache.append(k, v, off, st, tb, rows=3, sequences=3, max_pages=8, layer=layer, q=q, q_out=qo, heads=heads,
                     rope=rope, rope_positions=256)
        cache.attend(qo, ln, tb, out, heads=heads, sequences=3, max_pages=8, layer=layer)

    graph = None
    if capture:
        device.sync()
        device.capture_begin()
        launches()
        graph = device.capture_end()
    for step in range(6):
        if step == 3:  # one sequence ends, the rest move together
            pages.free(seqs[1])
            seqs[1] = seqs[0]  # (its place: a sequence of no rows of its own, below)
            pages.compact()
        live = [0, 2] if step >= 3 else [0, 1, 2]
        starts, lengths = [0xFFFFFF00] * 3, [0] * 3  # a place without a sequence: no position, no length
        for i in live:
            starts[i] = pages.grow(seqs[i], 1)
            lengths[i] = starts[i] + 1
        copies = pages.take_copies()
        if len(copies):
            cache.copy_pages(up(copies), len(copies))
        hq, hk, hv = rows(3, heads), rows(3, kv), rows(3, kv)
        for buf, x in ((q, hq), (k, hk), (v, hv), (st, np.array(starts, np.uint32)), (ln, np.array(lengths, np.uint32)),
                       (tb, pages.table(seqs, 8))):
            device.write(buf, x)
            device.sync()
        if graph:
            graph.launch()
        else:
            launches()
        got = device.read_array(out, np.float32, hq.size).reshape(hq.shape)
        for i in range(3):
            if i not in live:
                assert not got[i].any()
                continue
            s, p = seqs[i], starts[i]
            kr = rotate(hk[i:i + 1], cs[p:p + 1])
            rows_of[s] = tuple(np.concatenate([x, held(y)]) for x, y in zip(rows_of[s], (kr, hv[i:i + 1])))
            qr = rotate(hq[i:i + 1], cs[p:p + 1])[0].astype(np.float64)
            seen = np.ones(p + 1, bool)
            want = attend(qr, *rows_of[s], scale, seen)
            assert np.all(np.abs(got[i] - want) <= decode_bound(qr, *rows_of[s], scale, seen, want, "f32")), (step, i)
    if graph:
        graph.destroy()
    device.sync()
    cache.release()


def test_serving_run(device, up):
    serve(device, up, np.random.default_rng(31), capture=False)


def test_serving_run_captured(device, up):
    serve(device, up, np.random.default_rng(32), capture=True)


def test_two_captured_graphs_share_the_workspace(device, up):
    """Both split their keys, so both leave partials in the context's workspace; launched in turn, with
    an eager call between."""
    rng = np.random.default_rng(33)
    heads, kv, d, page, n = 4, 1, 64, 64, 3000
    P, k, v = random_pages(rng, 50, kv, d, page)
    cache = kv4.Kv4Cache(device, kv, d, 50, page, pool=up(P.pool))
    graphs = []
    for i in range(2):
        table = rng.permutation(50).astype(np.uint32)[None]
        q = rng.standard_normal((1, heads, d)).astype(np.float32)
        bq, bt, bl, out = up(q), up(table), up(np.array([n - 700 * i], np.uint32)), up(q.nbytes)
        device.capture_begin()
        cache.attend(bq, bl, bt, out, heads=heads, sequences=1, max_pages=50)
        g = device.capture_end()
        eager = up(q.nbytes)
        cache.attend(bq, bl, bt, eager, heads=heads, sequences=1, max_pages=50)
        graphs.append((g, out, device.read_array(eager, np.float32, q.size)))
    for turn in range(3):
        for g, out, want in graphs:
            g.launch()
        for g, out, want in graphs:
            np.testing.assert_array_equal(device.read_array(out, np.float32, want.size), want)
    for g, _, _ in graphs:
        g.destroy()


def test_on_a_callers_stream(device, up):
    """Launches go to the stream that the context is given (another context's here, which has work of its
    own on it before and after), and results are the same to the bit."""
    rng = np.random.default_rng(34)
    owner = K.Device(0)
    dev = K.Device(0, stream=owner.stream)
    assert dev.stream == owner.stream != device.stream
    q, k, v = (rng.standard_normal((2000, 4, 64)).astype(np.float16) for _ in range(3))
    off = up(np.array([0, 1200, 2000], np.uint32))
    bq, bk, bv, out, first, want = up(q.nbytes), up(k), up(v), up(q.nbytes), up(q.nbytes), up(q.nbytes)
    dims = dict(sequences=2, rows=2000, key_rows=2000, heads=4, kv_heads=4, head_dim=64)
    device.sync()
    kv4.attention_packed(owner, up(q), bk, bv, first, off, off, **dims)
    owner.write(bq, q)  # (on the stream, before the launch that reads it)
    kv4.attention_packed(dev, bq, bk, bv, out, off, off, **dims)
    owner.zero(bq, q.nbytes)
    got = dev.read_array(out, np.uint16, q.size)
    kv4.attention_packed(device, up(q), bk, bv, want, off, off, **dims)
    np.testing.assert_array_equal(got, device.read_array(want, np.uint16, q.size))
    assert got.any()
    dev.sync()
    dev.close()
    owner.close()
