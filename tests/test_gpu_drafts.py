"""The operators of a speculative step against their definitions in float64 (drafts_reference.py): tables within
their roundings, rotations and kept rows bit for bit, accepted branches and tokens exactly, the tree attention within
the decode attention's bounds (test_gpu_kv4.py), which count its roundings: the products, weights and sums are
the same, over at most as many positions. (Where columns share tiles 16-bit rows' weights are scaled by 2^12, not 2^15, and a
row's scores by its largest one and not by the group's scale: the first is 2^-37 of the largest weight for 2^-40, which the
2^-11 of every weight covers wherever the large weights' values are not 0; the second is one rounding less.)

A table's entry is one f32 rounding, 2^-24 of it, of amplitude (cos, sin) of an angle in 64 bits; a frequency is a few
64-bit operations (of 2^-53 each, a power one last place), so angles of both sides are within 16 x 2^-53 of themselves,
and the functions' own errors within 2^-51 on each side. Seven of eight positions are made from the one before by a product
of complex numbers of length 1: four products and sums of 2^-53 each, and the step's own 2^-51 in both of its parts, so up to
2^-53 (2 sqrt 2) + 2^-51 sqrt 2 < 2^-50 more with each, 7 x 2^-50 in all. A step's angle is off by 16 x 2^-53 of itself, seven
of them by less than 112 x 2^-53 of a step of at most 1: 2^-46 in all, which is 2^-22 of a table entry's f32 rounding.
"""

import ctypes

import numpy as np
import pytest

from drafts_reference import NO_ROW, frequencies, keep, rotate, tree_attend, verify_all
from enargeia_amd import _lib, drafts, kv4
from enargeia_amd import kernels as K
from kv4_reference import NO_PAGE, Pages, as_type, from_type, held, random_pages
from test_gpu_kv4 import decode_bound, kv4_size, offsets_of, tables, up  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def random_tree(rng, n, back=4):
    return np.array([-1] + [int(rng.integers(max(0, i - back), i)) for i in range(1, n)], np.int64).astype(np.uint32)[:n]


# ---- rotary positions ---------------------------------------------------------------------------------


@pytest.mark.parametrize("scaling", list(drafts.SCALINGS))
@pytest.mark.parametrize("positions,first,rotary", [(1, 0, 64), (300, 0, 8), (77, 131000, 128), (5, 2 ** 31 - 5, 24), (40, 12345, 512)])
def test_table(device, up, scaling, positions, first, rotary):  # noqa: F811
    print(f"table of {positions} from {first}, {rotary}, {scaling}", flush=True)
    how = dict(theta=5e5, factor=4.0, context=4096.0, low=1.5, high=20.0)
    out = up(np.full(positions * rotary + 64, 7.0, np.float32))
    drafts.rope_table(device, out, positions=positions, rotary_dim=rotary, first=first, scaling=scaling, amplitude=1.25, **how)
    got = device.read_array(out, np.float32, positions * rotary + 64)
    assert np.all(got[positions * rotary:] == 7.0)
    got = got[: positions * rotary].reshape(positions, rotary // 2, 2)
    angle = (first + np.arange(positions, dtype=np.float64))[:, None] * frequencies(rotary, scaling=scaling, **how)
    want = 1.25 * np.stack([np.cos(angle), np.sin(angle)], -1)
    bound = 2.0 ** -24 * np.abs(want) + 1.25 * (np.abs(angle) * 16 * 2.0 ** -53 + 2.0 ** -46)[..., None] * (1 + 2.0 ** -20)
    assert np.all(np.abs(got - want) <= bound)


def check_rope(device, up, rng, lengths, starts, depths, heads, kv, d, rotary, layout, in_type, out_type, before=0,  # noqa: F811
               after=0, pad=0, positions_in_table=None, in_place=False):
    rows = before + sum(lengths) + after
    within = np.concatenate([np.arange(n) for n in lengths]) if depths is None else depths
    position = np.repeat(starts, lengths) + within
    reach = int(position.max()) + 1 if positions_in_table is None else positions_in_table
    angle = np.arange(reach)[:, None] * 1e4 ** (-np.arange(0, rotary, 2) / rotary)
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    width = {"q": heads * d, "k": kv * d}
    x = {n: rng.standard_normal((rows, w + (pad if w else 0))).astype(np.float32) for n, w in width.items()}
    raw = {n: as_type(a, in_type) for n, a in x.items()}
    mark = 0x5A
    buf = {n: up(raw[n][0]) if x[n].size else None for n in x}
    outs = buf if in_place else {n: up(np.full((rows, x[n].shape[1] * kv4_size(out_type)), mark, np.uint8)) if x[n].size else None for n in x}
    p = None
    if depths is not None:
        p = up(np.concatenate([np.zeros(before, np.uint32), np.asarray(depths, np.uint32), np.zeros(after, np.uint32)]))
    stride = lambda n: x[n].shape[1] if pad else 0  # noqa: E731
    drafts.rope(device, up(cs), rows=rows, head_dim=d, rotary_dim=rotary, table_positions=reach, q=buf["q"], q_out=outs["q"],
                heads=heads, k=buf["k"], k_out=outs["k"], kv_heads=kv, positions=p, offsets=up(offsets_of(lengths, before)),
                starts=up(np.array(starts, np.uint32)), sequences=len(lengths), layout=layout, in_type=in_type,
                out_type=out_type, q_stride=stride("q"), k_stride=stride("k"), q_out_stride=stride("q"),
                k_out_stride=stride("k"))
    live = np.flatnonzero(position < reach)
    for n, w in width.items():
        if not w:
            continue
        v = np.asarray(raw[n][1], np.float32)
        want = np.frombuffer(np.ascontiguousarray(raw[n][0]).tobytes(), np.uint8).reshape(rows, -1).copy() if in_place else \
            np.full((rows, x[n].shape[1] * kv4_size(out_type)), mark, np.uint8)
        turned = rotate(v[before + live, :w].reshape(len(live), -1, d), cs[position[live]], rotary, layout)
        want[before + live, : w * kv4_size(out_type)] = np.ascontiguousarray(
            as_type(turned.reshape(len(live), w), out_type)[0]).view(np.uint8)
        got = device.read_array(outs[n], np.uint8, want.size).reshape(want.shape)
        np.testing.assert_array_equal(got, want, err_msg=n)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv,d,rotary", [(14, 2, 64, 64), (4, 1, 128, 64), (3, 3, 24, 8), (2, 0, 512, 512), (0, 5, 8, 8),
                                               (9, 1, 136, 120)])
def test_rope(device, up, layout, heads, kv, d, rotary):  # noqa: F811
    print(f"rope {heads}/{kv} x {d}, {rotary} {layout}", flush=True)
    rng = np.random.default_rng(heads + d)
    check_rope(device, up, rng, [1], [0], None, heads, kv, d, rotary, layout, "f32", "f32")
    check_rope(device, up, rng, [5, 0, 33, 1], [7, 9, 0, 100], None, heads, kv, d, rotary, layout, "f32", "f16", before=3, after=2)
    check_rope(device, up, rng, [4, 2], [50, 0], np.array([0, 1, 1, 2, 0, 1]), heads, kv, d, rotary, layout, "bf16", "f32", pad=8)


@pytest.mark.parametrize("in_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
def test_rope_types(device, up, in_type, out_type):  # noqa: F811
    for layout in drafts.LAYOUTS:
        check_rope(device, up, np.random.default_rng(5), [70, 3], [5, 0], None, 3, 2, 64, 48, layout, in_type, out_type)
    if in_type == out_type:
        for layout in drafts.LAYOUTS:
            check_rope(device, up, np.random.default_rng(6), [9], [5], None, 3, 2, 64, 48, layout, in_type, out_type, in_place=True, pad=8)


def test_rope_positions_past_the_table_and_many_sequences(device, up):  # noqa: F811
    rng = np.random.default_rng(7)
    check_rope(device, up, rng, [40], [20], None, 2, 1, 64, 64, "half", "f32", "f32", positions_in_table=50)
    check_rope(device, up, rng, [2, 2], [0xFFFFFFF0, 3], np.array([0, 0xFFFFFFFF, 1, 0]), 2, 1, 64, 64, "half", "f32", "f32",
               positions_in_table=50)
    lengths = [int(n) for n in rng.integers(0, 4, 200)]
    check_rope(device, up, rng, lengths, [int(s) for s in rng.integers(0, 40, 200)], None, 2, 1, 64, 32, "interleaved", "f32", "f16")
    check_rope(device, up, rng, [4000, 1], [0, 3], None, 14, 2, 64, 64, "half", "f16", "f16", before=1)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_of_q_and_k_in_one_buffer_in_place(device, up, layout):  # noqa: F811
    """Rows of q, k and v side by side, as one projection makes them: q and k rotated where they lie, v as it was."""
    rng = np.random.default_rng(12)
    rows, heads, kv, d = 37, 5, 2, 64
    x = rng.standard_normal((rows, (heads + 2 * kv) * d)).astype(np.float32)
    p = rng.integers(0, 90, rows).astype(np.uint32)
    angle = np.arange(90)[:, None] * 1e4 ** (-np.arange(0, d, 2) / d)
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    b = up(x)
    q, k, wide = K.Binding(b, 0), K.Binding(b, heads * d * 4), x.shape[1]
    drafts.rope(device, up(cs), rows=rows, head_dim=d, table_positions=90, q=q, q_out=q, heads=heads, k=k, k_out=k, kv_heads=kv, positions=up(p),
                layout=layout, q_stride=wide, k_stride=wide, q_out_stride=wide, k_out_stride=wide)
    want = x.copy()
    want[:, : (heads + kv) * d] = rotate(x[:, : (heads + kv) * d].reshape(rows, -1, d), cs[p], d, layout).reshape(rows, -1)
    np.testing.assert_array_equal(device.read_array(b, np.float32, x.size).reshape(x.shape), want)


def test_rope_without_sequences_and_without_starts(device, up):  # noqa: F811
    rng = np.random.default_rng(8)
    x, p = rng.standard_normal((6, 2, 64)).astype(np.float32), np.array([4, 0, 9, 2, 2, 10], np.uint32)
    angle = np.arange(10)[:, None] * 1e4 ** (-np.arange(0, 64, 2) / 64)
    cs = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
    b, t, out = up(x), up(cs), up(np.full(x.shape, 3.0, np.float32))
    common = dict(rows=6, head_dim=64, table_positions=10, q=b, q_out=out, heads=2)
    drafts.rope(device, t, positions=up(p), **common)
    want = np.full(x.shape, 3.0, np.float32)
    want[:5] = rotate(x[:5], cs[p[:5]], 64, "half")
    np.testing.assert_array_equal(device.read_array(out, np.float32, x.size).reshape(x.shape), want)
    drafts.rope(device, t, offsets=up(np.array([1, 4], np.uint32)), sequences=1, **common)
    want[1:4] = rotate(x[1:4], cs[:3], 64, "half")
    np.testing.assert_array_equal(device.read_array(out, np.float32, x.size).reshape(x.shape), want)


@pytest.mark.parametrize("d", [64, 128])
def test_rope_is_the_appends(device, up, d):  # noqa: F811
    """The same rows rotated by the append, by the same table: the same bits."""
    rng = np.random.default_rng(9)
    q, k = rng.standard_normal((9, 4, d)).astype(np.float32), rng.standard_normal((9, 2, d)).astype(np.float32)
    t = up(40 * d * 4)
    drafts.rope_table(device, t, positions=40, rotary_dim=d, theta=1e6)
    cache = kv4.Kv4Cache(device, 2, d, 1, 64)
    off, st, tb, bq, bk = up(np.array([0, 9], np.uint32)), up(np.array([30], np.uint32)), up(np.zeros(1, np.uint32)), up(q), up(k)
    a, b = ([up(q.nbytes), up(k.nbytes)] for _ in range(2))
    cache.append(bk, bk, off, st, tb, rows=9, sequences=1, max_pages=1, q=bq, q_out=a[0], k_out=a[1], heads=4, rope=t, rope_positions=40)
    drafts.rope(device, t, rows=9, head_dim=d, table_positions=40, q=bq, q_out=b[0], heads=4, k=bk, k_out=b[1], kv_heads=2,
                offsets=off, starts=st, sequences=1)
    for x, y, n in zip(a, b, (q.size, k.size)):
        np.testing.assert_array_equal(device.read_array(x, np.uint32, n), device.read_array(y, np.uint32, n))
    device.sync()
    cache.release()


# ---- the tree attention -------------------------------------------------------------------------------


def check_tree(device, up, rng, ns, lengths, heads, kv, d, page, kind, chain=False, extra=0, pad=0, scale=0.0, hole=None,  # noqa: F811
               before=0, after=0, q_of=None, max_rows=None, spread=1.0, parents=None, floor=0.0, step=1):
    """`floor`: of a weight's rounding, relative to the largest weight, where it is more than the decode's. Every step-th
    sequence is checked.

    An f16 output below 2^-14 is a multiple of 2^-24, so its rounding is off by up to 2^-25 whatever its size: a head whose large
    weights' values are 0 has such (weights 0.999995, 2.9e-6 and 2.1e-6 of values 0, -0.48 and 0.33 give -6.9e-7, between
    the numbers -12 x 2^-24 and -11 x 2^-24)."""
    pages = sum(-(-n // page) for n in lengths) + 1
    width = max(-(-n // page) for n in lengths) + 1 + extra
    P, kv_k, kv_v = random_pages(rng, pages, kv, d, page, spread)
    table = tables(rng, lengths, page, pages, width)
    for i, n in enumerate(lengths):  # beyond each sequence's end its last page holds scales that are no numbers
        if n % page:
            for h in range(kv):
                _, _, ks, vs = P._streams(table[i, n // page], h)
                ks[:, n % page:] = np.nan
                vs[:, n % page:] = np.inf
    if hole is not None:
        table[hole] = pages  # a page that is none
    rows = before + sum(ns) + after
    q = rng.standard_normal((rows, heads * d + pad)).astype(np.float32) if q_of is None else q_of
    raw, val = as_type(q, kind)
    if parents is None and not chain:
        parents = np.concatenate([np.full(before, 7, np.uint32)] + [random_tree(rng, n) for n in ns] + [np.full(after, 7, np.uint32)])
    out = up(np.full((rows, (heads * d + pad) * kv4_size(kind)), 0x5A, np.uint8))
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(P.pool))
    off = offsets_of(ns, before)
    cache.attend_tree(up(raw), up(off), up(np.array(lengths, np.uint32)), up(table), out, parents=None if chain else up(parents),
                      heads=heads, rows=rows, max_rows=max_rows or max(ns + [1]), sequences=len(ns), max_pages=width, type=kind,
                      scale=scale, q_stride=heads * d + pad if pad else 0, out_stride=heads * d + pad if pad else 0)
    size = kv4_size(kind)
    bytes_ = device.read_array(out, np.uint8, q.size * size).reshape(rows, -1)
    got = from_type(bytes_.tobytes(), kind).reshape(q.shape)
    assert np.all(bytes_[:, heads * d * size:] == 0x5A)
    assert np.all(bytes_[:before] == 0x5A) and np.all(bytes_[rows - after:] == 0x5A)
    f = scale or 1.0 / np.sqrt(d)
    for i, (n, length) in list(enumerate(zip(ns, lengths)))[::step]:
        r = slice(int(off[i]), int(off[i + 1]))
        ids = table[i, : -(-length // page)]
        have = (np.repeat(ids, page) < pages)[:length]
        ids = np.minimum(ids, pages - 1)
        k, v = (x[ids].reshape(-1, kv, d)[:length] for x in (kv_k, kv_v))
        qi = val[r, : heads * d].reshape(n, heads, d)
        want, seen = tree_attend(qi, k, v, f, None if chain else parents[r], have) if n else (np.zeros((0, heads, d)), None)
        for j in range(n):
            bound = decode_bound(qi[j], k, v, f, seen[j], want[j], kind) + floor * seen[j].sum() * np.abs(v).max()
            bound = bound + (2.0 ** -25 if kind == "f16" else 0.0)
            off_by = np.abs(got[r][j, : heads * d].reshape(heads, d) - want[j])
            assert np.all(off_by <= bound), (f"row {j} of {n}, sequence {i} of {length}: off by {np.nanmax(off_by / bound):.2f} of the "
                                             f"bound", kind)
    return got


LAYOUTS = [(14, 2, 64, 64), (8, 8, 64, 32), (12, 4, 64, 256), (16, 1, 128, 128), (8, 2, 128, 32), (40, 2, 64, 64)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,page", LAYOUTS)
def test_tree_rows_and_lengths(device, up, heads, kv, d, page, kind):  # noqa: F811
    print(f"tree {heads}/{kv} x {d}, page {page}, {kind}", flush=True)
    rng = np.random.default_rng(heads + d)
    ns, lengths = [1, 5, 16, 2, 0, 33, 64, 17], [1, 5, 400, 300, 9, 66, 130, 31]
    check_tree(device, up, rng, ns, lengths, heads, kv, d, page, kind, before=2, after=3)
    check_tree(device, up, rng, [4, 1, 64], [4, 257, 96], heads, kv, d, page, kind, chain=True)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 31, 32, 33, 47, 48, 63, 64])
def test_tree_every_number_of_rows_at_every_place_in_a_tile(device, up, n):  # noqa: F811
    rng = np.random.default_rng(n)
    lengths = [n, n + 1, n + 15, n + 31, n + 32, 64 + n // 2, max(n, 96), max(n, 97), 128 + n]
    check_tree(device, up, rng, [n] * len(lengths), lengths, 4, 2, 64, 32, "f32")
    check_tree(device, up, rng, [n] * len(lengths), lengths, 3, 1, 128, 64, "bf16")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,d", [(14, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("ns,lengths,extra", [([20], [3000], 0), ([3], [5], 50), ([9], [513], 60), ([5, 1, 0, 64], [2500, 40, 9, 1111], 3)])
def test_tree_splits(device, up, heads, kv, d, ns, lengths, extra, kind):  # noqa: F811
    check_tree(device, up, np.random.default_rng(sum(lengths)), ns, lengths, heads, kv, d, 64, kind, extra=extra)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_tree_strides_scale_and_holes(device, up, kind):  # noqa: F811
    rng = np.random.default_rng(3)
    check_tree(device, up, rng, [6, 20], [200, 130], 6, 2, 64, 32, kind, pad=16, scale=0.3, hole=(0, 2))
    check_tree(device, up, rng, [6, 20], [200, 130], 6, 2, 128, 32, kind, pad=8, hole=(1, 4))  # the rows' own last page
    check_tree(device, up, rng, [40], [40], 2, 1, 64, 32, kind, hole=(0, 0))  # rows that see nothing, or only some of theirs
    check_tree(device, up, rng, [5, 7], [5, 7], 2, 1, 64, 32, kind, hole=(slice(None), slice(None)))


def test_tree_many_sequences(device, up):  # noqa: F811
    rng = np.random.default_rng(4)
    ns = [int(n) for n in rng.integers(0, 9, 150)]
    check_tree(device, up, rng, ns, [n + int(x) for n, x in zip(ns, rng.integers(0, 60, 150))], 4, 2, 64, 32, "f16", max_rows=64)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d,page,n,length,seqs", [(4, 64, 64, 4, 9000, 300), (2, 128, 32, 5, 8600, 300), (8, 64, 32, 6, 2500, 300),
                                                        (16, 128, 64, 3, 4300, 300), (16, 64, 64, 7, 4300, 300),
                                                        (16, 128, 256, 8, 2300, 300), (4, 64, 64, 4, 17500, 256), (16, 64, 64, 16, 2500, 256),
                                                        (16, 128, 32, 16, 4300, 256)])
def test_tree_chunks_of_more_steps_than_a_wave_holds_page_ids(device, up, heads, d, page, n, length, seqs, kind):  # noqa: F811
    """As many sequences as CUs or more, so that none is split, over the same pages: every kernel past the page ids that a wave reads at
    once. Some of the sequences are checked."""
    rng = np.random.default_rng(length + d)
    pages = -(-length // page)
    P, k, v = random_pages(rng, pages, 1, d, page)
    order = rng.permutation(pages).astype(np.uint32)
    kk, vv = (x[order].reshape(-1, 1, d) for x in (k, v))
    lengths = rng.integers(length - 600, length + 1, seqs).astype(np.uint32)
    lengths[:2] = length, n
    parents = np.concatenate([random_tree(rng, n) for _ in range(seqs)])
    raw, val = as_type(rng.standard_normal((seqs * n, heads * d)).astype(np.float32), kind)
    out = up(raw.nbytes)
    cache = kv4.Kv4Cache(device, 1, d, pages, page, pool=up(P.pool))
    cache.attend_tree(up(raw), up(offsets_of([n] * seqs)), up(lengths), up(np.tile(order, (seqs, 1))), out, parents=up(parents),
                      heads=heads, rows=seqs * n, max_rows=n, sequences=seqs, max_pages=pages, type=kind)
    got = from_type(device.read(out, raw.nbytes), kind).reshape(seqs, n, heads, d)
    for s in (0, 1, 2, seqs - 1):
        m = int(lengths[s])
        q = val.reshape(seqs, n, heads, d)[s]
        want, seen = tree_attend(q, kk[:m], vv[:m], d ** -0.5, parents[s * n:(s + 1) * n], np.ones(m, bool))
        for j in range(n):
            bound = decode_bound(q[j], kk[:m], vv[:m], d ** -0.5, seen[j], want[j], kind)
            assert np.all(np.abs(got[s, j] - want[j]) <= bound), (s, j, float(np.max(np.abs(got[s, j] - want[j]) / bound)))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,page,n,extra,seqs", [(64, 32, 8, 12, 36), (64, 64, 16, 4, 36), (64, 128, 40, 2, 36), (128, 32, 8, 12, 36),
                                                 (128, 256, 16, 1, 36), (128, 64, 40, 5, 36), (128, 32, 16, 90, 36),
                                                 (64, 64, 32, 8, 32), (128, 32, 32, 24, 32)])
def test_tree_many_columns_and_sequences(device, up, d, page, n, extra, seqs, kind):  # noqa: F811
    """Enough columns and sequences that they share tiles (64, 128 and 256 a workgroup), at every place in a step; tables that reach
    far past the lengths; pages that are none under the rows and before them. 16-bit rows' weights are scaled by 2^12 at least, of
    which half a step of f16's smallest numbers, 2^-25, is 2^-37."""
    floor = 0.0 if kind == "f32" else 2.0 ** -37
    rng = np.random.default_rng(d + n + extra)
    ns = [n if i % 5 == 0 else int(rng.integers(0, n + 1)) for i in range(seqs)]
    places = [0, 1, 15, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 130]
    lengths = [max(1, k + places[i % len(places)]) for i, k in enumerate(ns)]
    lengths[0] = 330
    hole = ([0, 4, 10], [1 if page < 256 else 0, 0, 0])
    check_tree(device, up, rng, ns, lengths, 64, 8, d, page, kind, extra=extra, hole=hole, before=1, after=2, floor=floor, step=2)
    check_tree(device, up, rng, ns, lengths, 64, 8, d, page, kind, extra=extra, chain=True, pad=8, scale=0.7, floor=floor, step=5)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("d,n,length,seqs", [(64, 8, 500, 36), (64, 16, 40, 36), (64, 40, 200, 36), (128, 8, 450, 36), (128, 16, 47, 36),
                                             (128, 40, 300, 36), (64, 32, 480, 32), (128, 32, 700, 32)])
def test_tree_not_finite_rows_where_columns_share_tiles(device, up, d, n, length, seqs, kind):  # noqa: F811
    """As test_tree_not_finite_rows_stay_with_who_sees_them, in one of many sequences over one table: the others, whose rows lie
    in other pages, keep their bits."""
    rng = np.random.default_rng(n + d)
    heads, kv, page = 64, 8, 32
    parents = random_tree(rng, n, 5)
    each = -(-length // page)
    whole = (length - n) // page  # the pages of no sequence's rows are shared
    pages = whole + seqs * (each - whole)
    P, k, v = random_pages(rng, pages, kv, d, page)
    table = np.zeros((seqs, each + 12), np.uint32)
    table[:, :whole] = np.arange(whole)
    table[:, whole:each] = whole + rng.permutation(pages - whole).reshape(seqs, -1)
    q = rng.standard_normal((seqs * n, heads, d)).astype(np.float32)
    raw, _ = as_type(q, kind)
    off, ln, tb, bq, pr, out = (up(x) for x in (offsets_of([n] * seqs), np.full(seqs, length, np.uint32), table, raw, np.tile(parents, seqs), raw))
    bad_seq, bad_head = 17, 5
    clean = None
    for what, row, group in [(None, 0, 0), ("v", n // 2, 0), ("v", 1, d // 32 - 1), ("k", n // 2, 1), ("v", n - 1, 1), ("v", 0, 0)]:
        pool = Pages(pages, kv, d, page)
        pool.pool[:] = P.pool
        if what:
            p = length - n + row
            _, _, ks, vs = pool._streams(table[bad_seq, p // page], bad_head)
            (ks if what == "k" else vs)[group, p % page] = np.nan
        cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(pool.pool))
        cache.attend_tree(bq, off, ln, tb, out, parents=pr, heads=heads, rows=seqs * n, max_rows=n, sequences=seqs,
                          max_pages=each + 12, type=kind)
        got = from_type(device.read(out, raw.nbytes), kind).reshape(seqs, n, kv, heads // kv, d)
        if what is None:
            clean = got
            assert np.all(np.isfinite(clean))
            continue
        bad = np.zeros(got.shape, bool)
        for i in range(n):
            j = i
            while j != row and int(parents[j]) < j:
                j = int(parents[j])
            if j == row:
                bad[bad_seq, i, bad_head, :, 32 * group if what == "v" else 0: 32 * (group + 1) if what == "v" else d] = True
        np.testing.assert_array_equal(np.isnan(got), bad, err_msg=f"{what} of row {row}")
        np.testing.assert_array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,d,n,length", [(128, 1, 64, 64, 150), (96, 1, 128, 37, 600), (1, 1, 128, 1, 1), (33, 33, 64, 2, 70)])
def test_tree_of_the_most_and_fewest_columns(device, up, heads, kv, d, n, length, kind):  # noqa: F811
    """8,192 columns of a kv head, and one; 16-bit rows' weights as in test_tree_many_columns_and_sequences."""
    rng = np.random.default_rng(heads)
    check_tree(device, up, rng, [n, max(1, n // 3)], [length, length], heads, kv, d, 32, kind, floor=0.0 if kind == "f32" else 2.0 ** -37)


def test_tree_parents_that_are_none(device, up):  # noqa: F811
    """Parents that are not before their row: such rows are roots, and see no other row."""
    rng = np.random.default_rng(5)
    parents = np.array([3, 0, 2, 9, 3, 0xFFFFFFFF, 5], np.uint32)
    check_tree(device, up, rng, [7], [50], 4, 2, 64, 32, "f32", parents=parents)


@pytest.mark.parametrize("kind,factor", [("f32", 0.0), ("f32", 1e-30), ("f16", 1e-4), ("f32", 40.0), ("bf16", 300.0)])
def test_tree_query_sizes(device, up, factor, kind):  # noqa: F811
    rng = np.random.default_rng(6)
    q = (rng.standard_normal((27, 4 * 64)) * factor).astype(np.float32)
    check_tree(device, up, rng, [7, 20], [300, 64], 4, 2, 64, 64, kind, q_of=q)


def test_tree_of_one_row_is_the_decode(device, up):  # noqa: F811
    """A chain of one row is the decode attention's case: both within the bounds, and of the same values."""
    rng = np.random.default_rng(7)
    P, k, v = random_pages(rng, 12, 2, 64, 64)
    cache = kv4.Kv4Cache(device, 2, 64, 12, 64, pool=up(P.pool))
    q, lengths = rng.standard_normal((2, 14, 64)).astype(np.float32), [333, 70]
    table = tables(rng, lengths, 64, 12, 6)
    b, ln, tb, a, c = up(q), up(np.array(lengths, np.uint32)), up(table), up(q.nbytes), up(q.nbytes)
    cache.attend(b, ln, tb, a, heads=14, sequences=2, max_pages=6)
    cache.attend_tree(b, up(np.array([0, 1, 2], np.uint32)), ln, tb, c, heads=14, rows=2, max_rows=1, sequences=2, max_pages=6)
    x, y = (device.read_array(o, np.float32, q.size).reshape(q.shape) for o in (a, c))
    for i, n in enumerate(lengths):
        ids = table[i, : -(-n // 64)]
        kk, vv = (z[ids].reshape(-1, 2, 64)[:n] for z in (k, v))
        seen = np.ones(n, bool)
        bound = decode_bound(q[i].astype(np.float64), kk, vv, 0.125, seen, x[i].astype(np.float64), "f32")
        assert np.all(np.abs(x[i].astype(np.float64) - y[i]) <= 2 * bound)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,length", [(9, 9), (9, 40), (40, 75), (64, 700)])
def test_tree_not_finite_rows_stay_with_who_sees_them(device, up, n, length, d):  # noqa: F811
    """A row whose K or V is no number, in one group of dims of one head: those below it have NaN, in V's case in
    that group of dims; the others are as ever."""
    rng = np.random.default_rng(n + d)
    heads, kv, page = 6, 2, 32
    parents = random_tree(rng, n, 5)
    pages = -(-length // page)
    P, k, v = random_pages(rng, pages, kv, d, page)
    table = rng.permutation(pages).astype(np.uint32)[None]
    q = rng.standard_normal((n, heads, d)).astype(np.float32)
    off, ln, tb, bq, pr, out = (up(x) for x in (np.array([0, n], np.uint32), np.array([length], np.uint32), table, q, parents, q))
    clean = None
    for what, row, group in [(None, 0, 0), ("v", n // 2, 0), ("v", 1, d // 32 - 1), ("k", n // 2, 1), ("v", n - 1, 1)]:
        pool = Pages(pages, kv, d, page)
        pool.pool[:] = P.pool
        if what:
            p = length - n + row
            _, _, ks, vs = pool._streams(table[0, p // page], 1)
            (ks if what == "k" else vs)[group, p % page] = np.nan
        cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(pool.pool))
        cache.attend_tree(bq, off, ln, tb, out, parents=pr, heads=heads, rows=n, max_rows=n, sequences=1, max_pages=pages)
        got = device.read_array(out, np.float32, q.size).reshape(q.shape)
        if what is None:
            clean = got
            assert np.all(np.isfinite(clean))
            continue
        bad = np.zeros(got.shape, bool)
        for i in range(n):
            j = i
            while j != row and int(parents[j]) < j:
                j = int(parents[j])
            if j == row:
                bad[i, 3:, 32 * group if what == "v" else 0: 32 * (group + 1) if what == "v" else d] = True
        np.testing.assert_array_equal(np.isnan(got), bad, err_msg=f"{what} of row {row}")
        np.testing.assert_array_equal(got[~bad], clean[~bad])


def test_tree_lengths_that_do_not_fit(device, up):  # noqa: F811
    """Fewer positions than rows: zeros. More rows than max_rows, offsets past the rows or descending: not written. A
    length past the table: what the table has of the positions before the rows."""
    rng = np.random.default_rng(8)
    P, k, v = random_pages(rng, 2, 1, 64, 32)
    cache = kv4.Kv4Cache(device, 1, 64, 2, 32, pool=up(P.pool))
    q = rng.standard_normal((10, 4, 64)).astype(np.float32)
    bq, tb = up(q), up(np.array([[1, 0]] * 4, np.uint32))

    def run(off, lengths, max_rows=4, rows=10):
        out = up(np.full(q.shape, 9.0, np.float32))
        cache.attend_tree(bq, up(np.array(off, np.uint32)), up(np.array(lengths, np.uint32)), tb, out, heads=4, rows=rows,
                          max_rows=max_rows, sequences=len(lengths), max_pages=2)
        return device.read_array(out, np.float32, q.size).reshape(q.shape)

    got = run([0, 3, 8, 10], [2, 20, 0xFFFFFFFF])
    assert not got[:3].any() and np.all(got[3:8] == 9.0)
    kk, vv = (x[[1, 0]].reshape(-1, 1, 64) for x in (k, v))
    for r in (8, 9):
        want, seen = tree_attend(q[r:r + 1].astype(np.float64), np.concatenate([kk, kk[:1]]), np.concatenate([vv, vv[:1]]), 0.125,
                                 None, np.arange(65) < 64)
        bound = decode_bound(q[r].astype(np.float64), kk, vv, 0.125, np.ones(64, bool), want[0], "f32")
        assert np.all(np.abs(got[r] - want[0]) <= bound)
    for off in ([0, 3, 11], [0xFFFFFFFF, 2, 3], [5, 2, 3]):
        got = run(off, [30, 30])
        last = slice(off[1], off[2])
        ok = np.zeros(10, bool)
        if off[2] <= 10:
            ok[last] = True
        else:
            ok[:3] = True
        assert np.all(got[~ok] == 9.0) and np.all(got[ok] != 9.0)
    assert np.all(run([0, 3, 4], [30, 30], rows=3)[3:] == 9.0)


def test_tree_pool_past_4_gib(device, up):  # noqa: F811
    """Pages 128 MiB apart: attention and kept rows at byte offsets past 32 bits."""
    rng = np.random.default_rng(16)
    kv, d, page, stride, pages, n = 1, 64, 32, 1 << 27, 36, 12
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(stride * (pages - 1) + kv4.page_bytes(kv, d, page)))
    cache.dims.page_stride = stride
    x = rng.standard_normal((2, 40, d)).astype(np.float32)
    off, st, tb = up(np.array([0, 40], np.uint32)), up(np.zeros(1, np.uint32)), up(np.array([[34, 33]], np.uint32))
    cache.append(up(x[0]), up(x[1]), off, st, tb, rows=40, sequences=1, max_pages=2)
    q = rng.standard_normal((n, 3, d)).astype(np.float32)
    out, ro, ln, new = up(q.nbytes), up(np.array([0, n], np.uint32)), up(np.array([40], np.uint32)), up(4)
    cache.attend_tree(up(q), ro, ln, tb, out, heads=3, rows=n, max_rows=n, sequences=1, max_pages=2)
    got = device.read_array(out, np.float32, q.size).reshape(q.shape)
    k, v = held(x[0])[:, None], held(x[1])[:, None]
    want, seen = tree_attend(q.astype(np.float64), k, v, 0.125, None, np.ones(40, bool))
    for i in range(n):
        assert np.all(np.abs(got[i] - want[i]) <= decode_bound(q[i].astype(np.float64), k, v, 0.125, seen[i], want[i], "f32"))
    path = np.array([[0, 2, 3, 7, 11] + [NO_ROW] * 7], np.uint32)
    cache.keep(up(path), up(np.array([5], np.uint32)), ro, ln, tb, new, max_rows=n, sequences=1, max_pages=2)
    assert device.read_array(new, np.uint32, 1)[0] == 33
    ko, vo = up(33 * d * 4), up(33 * d * 4)
    cache.read(ko, vo, up(np.array([0, 33], np.uint32)), st, tb, rows=33, sequences=1, max_pages=2, out_type="f32")
    order = list(range(28)) + [28 + int(j) for j in path[0, :5]]
    np.testing.assert_array_equal(device.read_array(ko, np.float32, 33 * d).reshape(33, d), k[order, 0])
    np.testing.assert_array_equal(device.read_array(vo, np.float32, 33 * d).reshape(33, d), v[order, 0])


# ---- verification -------------------------------------------------------------------------------------


def check_verify(device, up, logits, tokens, ns, parents, draft, accept, draws, temperatures, kind="f32", before=0, after=0,  # noqa: F811
                 max_rows=None, pad=0):
    """`logits` [rows, vocab] etc. of the packed rows; rows before and after are put around them."""
    rows, vocab = logits.shape
    around = lambda a, fill: None if a is None else np.concatenate([np.full((before, *a.shape[1:]), fill, a.dtype), a,  # noqa: E731
                                                                    np.full((after, *a.shape[1:]), fill, a.dtype)])
    raw, val = as_type(np.pad(logits, ((0, 0), (0, pad)), constant_values=99.0), kind)
    off = offsets_of(ns, before)
    width = max_rows if max_rows is not None else max(ns + [1])
    s = len(ns)
    path, counts, token = up(np.full((s, width + 1), 5, np.uint32)), up(4 * s + 4), up(4 * s + 4)
    f32 = lambda a: None if a is None else np.asarray(a, np.float32)  # noqa: E731
    b = [None if a is None else up(a) for a in (around(raw, 0), around(np.asarray(tokens, np.uint32), 0), off,
                                                around(None if parents is None else np.asarray(parents, np.uint32), 0),
                                                around(None if draft is None else np.pad(f32(draft), ((0, 0), (0, pad))), 0),
                                                around(f32(accept), 0), f32(draws), f32(temperatures))]
    drafts.verify(device, b[0], b[1], b[2], path, counts, token, parents=b[3], draft=b[4], accept=b[5], draws=b[6],
                  temperatures=b[7], sequences=s, rows=before + rows + after, max_rows=width, vocab=vocab, type=kind,
                  logits_stride=vocab + pad if pad else 0, draft_stride=vocab + pad if pad else 0)
    got = (device.read_array(path, np.uint32, s * width).reshape(s, width), device.read_array(counts, np.uint32, s),
           device.read_array(token, np.uint32, s))
    want = verify_all(val[:, :vocab], tokens, off - before, parents, draft, f32(accept), f32(draws), f32(temperatures), width)
    for x, y, name in zip(got, want, ("path", "counts", "next")):
        np.testing.assert_array_equal(x, y, err_msg=name)
    return want


def verify_case(rng, ns, vocab, chain, with_draft, peak=6.0):
    """Logits with some likely tokens, and drafts that are often among them."""
    rows = sum(ns)
    x = rng.standard_normal((rows, vocab)) * 1.5
    x[np.arange(rows)[:, None], rng.integers(0, vocab, (rows, 3))] += peak * rng.random((rows, 3))
    parents = None if chain else np.concatenate([random_tree(rng, n, 3) for n in ns])
    first = np.repeat(np.cumsum([0] + ns[:-1]), ns)
    local = np.arange(rows) - first
    up_ = first + np.where(local == 0, 0, local - 1 if chain else np.minimum(np.concatenate([parents]) if not chain else 0, local))
    blurred = x + rng.standard_normal((rows, vocab)) * 0.5
    e = np.exp(blurred - blurred.max(-1, keepdims=True))
    q = (e / e.sum(-1, keepdims=True)).astype(np.float32)
    if with_draft:
        tokens = np.array([rng.choice(vocab, p=q[u] / q[u].astype(np.float64).sum()) for u in up_])
    else:  # the likeliest of the parent's row, siblings the next ones
        order = np.argsort(-blurred, -1)
        rank = [sum(1 for j in range(i) if up_[j] == up_[i] and local[j] > 0) for i in range(rows)]
        tokens = np.array([order[u, min(r, vocab - 1)] for u, r in zip(up_, rank)])
    return x.astype(np.float32), tokens, parents, q if with_draft else None


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 7, 300, 4096, 4097, 20011])
@pytest.mark.parametrize("how", ["greedy", "chain", "tree", "draft"])
def test_verify(device, up, vocab, how, kind):  # noqa: F811
    print(f"verify {how}, vocab {vocab}, {kind}", flush=True)
    rng = np.random.default_rng(vocab + len(how))
    for ns, before, after, pad in (([1], 0, 0, 0), ([5, 0, 1, 16], 2, 3, 0), ([64, 3, 33], 0, 1, 5)):
        x, tokens, parents, draft = verify_case(rng, ns, vocab, how in ("chain", "draft"), how == "draft")
        t = None if how == "greedy" else np.where(rng.random(len(ns)) < 0.8, rng.uniform(0.5, 1.5, len(ns)), 0.0)
        check_verify(device, up, x, tokens, ns, parents, draft, rng.random(sum(ns)), rng.random(len(ns)), t, kind, before, after,
                     64 if before else None, pad)


def test_verify_the_whole_vocabulary(device, up):  # noqa: F811
    """Of the package's own model: 38 chunks, the last one partial."""
    rng = np.random.default_rng(3)
    for chain, draft in ((True, True), (False, False)):
        ns = [4, 2]
        x, tokens, parents, q = verify_case(rng, ns, 151936, chain, draft, peak=14.0)
        for _ in range(3):
            check_verify(device, up, x, tokens, ns, parents, q, rng.random(6), rng.random(2), [0.9, 1.1])


@pytest.mark.parametrize("how", ["chain", "tree", "draft"])
@pytest.mark.parametrize("vocab,kind", [(1 << 20, "f32"), ((1 << 20) - 4097, "bf16")])
def test_verify_the_largest_vocabularies(device, up, vocab, kind, how):  # noqa: F811
    """256 and 255 chunks: a row's sums in four reads of a wave, a chunk a thread in the draw; the ends of what can be drawn."""
    rng = np.random.default_rng(vocab + len(how))
    ns = [3, 1]
    x, tokens, parents, q = verify_case(rng, ns, vocab, how != "tree", how == "draft", peak=14.0)
    one = np.nextafter(np.float32(1), np.float32(0))
    for draws in ([0.0, one], rng.random(2)):
        check_verify(device, up, x, tokens, ns, parents, q, rng.random(4), draws, [0.9, 1.3], kind)


def test_verify_draws_over_every_id(device, up):  # noqa: F811
    """Numbers from 0 to the largest below 1, of a flat row: every part of a chunk, and every chunk's ends."""
    rng = np.random.default_rng(4)
    vocab, s = 12289, 120
    x = np.tile(rng.standard_normal((1, vocab)).astype(np.float32) * 0.1, (s, 1))
    u = np.linspace(0, 1, s, endpoint=False).astype(np.float32)
    u[-1] = np.nextafter(np.float32(1), np.float32(0))
    want = check_verify(device, up, x, np.zeros(s, int), [1] * s, None, None, np.zeros(s), u, np.ones(s))
    assert want[2][0] == 0 and want[2][-1] >= vocab - 2 and len(set(want[2])) == s


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("how", ["chain", "tree", "draft"])
def test_verify_many_sequences(device, up, how, kind):  # noqa: F811
    """More chunks than are drawn from one a workgroup: four at a time, the last ones partial."""
    rng = np.random.default_rng(len(how))
    for vocab, s in ((20011, 260), (36864, 130)):
        ns = [int(n) for n in rng.integers(0, 3, s)]
        x, tokens, parents, draft = verify_case(rng, ns, vocab, how != "tree", how == "draft")
        t = np.where(rng.random(s) < 0.9, rng.uniform(0.5, 1.5, s), 0.0)
        check_verify(device, up, x, tokens, ns, parents, draft, rng.random(sum(ns)), rng.random(s), t, kind, 1, 2)


def test_verify_many_children_and_tokens_again(device, up):  # noqa: F811
    """63 children of a root: all rejected, the last accepted, the first; tokens that siblings had before; tokens that are no
    ids; the largest numbers."""
    rng = np.random.default_rng(5)
    vocab, n = 9000, 64
    x = (rng.standard_normal((n, vocab)) * 0.5).astype(np.float32)
    parents = np.array([0xFFFFFFFF] + [0] * 63, np.uint32)
    one = np.nextafter(np.float32(1), np.float32(0))
    tokens = rng.integers(0, vocab, n)
    tokens[10:20] = tokens[9]
    tokens[20:22] = [vocab, 0xFFFFFFFF]
    for accept in (np.full(n, one), np.where(np.arange(n) == 63, 0, one), np.zeros(n), np.where(np.arange(n) == 12, 0, one),
                   np.where((np.arange(n) == 20) | (np.arange(n) == 40), 0, one)):
        for draw in (0.0, 0.37, one):
            check_verify(device, up, x, tokens, [n], parents, None, accept, [draw], [1.0])
    x[0] = -30.0
    x[0, tokens[:40] % vocab] = rng.standard_normal(40)  # nearly all lies in the rejected ones
    check_verify(device, up, x, tokens % vocab, [n], parents, None, np.full(n, one), [0.5], [1.0])


def test_verify_masked_and_not_finite_logits(device, up):  # noqa: F811
    rng = np.random.default_rng(6)
    vocab, rows = 5000, 3
    base = rng.standard_normal((rows, vocab)).astype(np.float32)
    for fill, at in ((-np.inf, slice(0, 4999)), (-np.inf, slice(0, None)), (np.nan, slice(17, 18)), (np.inf, slice(4500, 4502)),
                     (np.nan, slice(0, None)), (-np.inf, slice(4000, None)), (-3.4e38, slice(1, None)), (3.4e38, slice(7, 9)),
                     (np.finfo(np.float32).min, slice(0, None))):
        for row in range(rows):
            x = base.copy()
            x[row, at] = fill
            for t in (0.0, 0.7):
                tokens = [0, 4999, 8]
                check_verify(device, up, x, tokens, [rows], None, None, [0, 1e-6, 0.0], [0.3], [t])
                q = np.full((rows, vocab), 1 / vocab, np.float32)
                check_verify(device, up, x, tokens, [rows], None, q, [0, 0.9, 0.9], [0.3], [t])


def test_verify_temperatures(device, up):  # noqa: F811
    """Small ones decide as greedy does, large ones draw from an even row; not above 0 is greedy."""
    rng = np.random.default_rng(7)
    x, tokens, parents, _ = verify_case(rng, [8] * 6, 3000, False, False)
    check_verify(device, up, x, tokens, [8] * 6, parents, None, rng.random(48), rng.random(6),
                 [1e-6, 1e-38, 1e30, -1.0, float("nan"), 2.5])
    check_verify(device, up, x, tokens, [8] * 6, parents, None, rng.random(48), rng.random(6), [9e-31, 1.1e-30, 1e-20, 1e38, 0.0, 0.01])


def test_verify_numbers_next_to_a_border(device, up):  # noqa: F811
    """Numbers that are p(x), and what p(x) is of what is left, to f32's rounding: just under, at and just over them. What a
    sum in f32 would say of them is a coin's toss; 64 bits decide by the numbers' own roundings, of 2^-25 and more."""
    rng = np.random.default_rng(9)
    vocab, n = 30001, 4
    x = (rng.standard_normal((n, vocab)) * 2).astype(np.float32)
    x[:, :50] += 6
    tokens, parents = np.array([0, 7, 33, 21]), np.array([9, 0, 0, 0], np.uint32)
    for t in (1.0, 0.73):
        t32 = np.float64(np.float32(t))
        e = np.exp((x[0].astype(np.float64) - x[0].max()) / t32)
        p = e / e.sum()
        one = np.float32(1) - np.float32(2.0 ** -24)
        for r, border in ((1, p[7]), (2, p[33] / (1 - p[7])), (3, p[21] / (1 - p[7] - p[33]))):
            u = np.float32(border)
            for number in (np.nextafter(u, np.float32(0)), u, np.nextafter(u, np.float32(1))):
                accept = np.where(np.arange(n) < r, one, np.float32(0.5))
                accept[r] = number
                check_verify(device, up, x, tokens, [n], parents, None, accept, [0.4], [t])
    # a chain: every row's number next to its border, so that several rows of a sequence are summed again
    tokens = np.array([0, 3, 8, 40])
    e = np.exp(x.astype(np.float64) - x.max(-1, keepdims=True))
    p = (e / e.sum(-1, keepdims=True))[np.arange(3), tokens[1:]]
    for down in (0, 1):
        accept = np.concatenate([[0], np.nextafter(np.float32(p), np.float32(1 - down))])
        check_verify(device, up, np.tile(x, (3, 1)), np.tile(tokens, 3), [4, 4, 4], None, None, np.tile(accept, 3), [0.1, 0.5, 0.9], [1.0] * 3)


def test_verify_equal_logits_go_to_the_lowest_id(device, up):  # noqa: F811
    x = np.zeros((4, 10000), np.float32)
    x[0, [4095, 4096, 9999]] = 2.0
    x[1, [256, 255]] = 2.0
    want = check_verify(device, up, x, [0, 4095, 256, 0], [4], None, None, None, None, None)
    assert want[0][0, :2].tolist() == [0, 1] and want[2][0] == 255


def test_verify_sequences_that_are_not_computed(device, up):  # noqa: F811
    rng = np.random.default_rng(8)
    x, tokens, parents, _ = verify_case(rng, [5, 0, 9, 2], 500, False, False)
    want = check_verify(device, up, x, tokens, [5, 0, 9, 2], parents, None, rng.random(16), rng.random(4), [1.0] * 4, max_rows=5)
    assert want[1][1] == want[1][2] == 0 and want[2][2] == NO_ROW and want[0].shape == (4, 5)
    # offsets past the rows, and descending ones
    b, t, u = up(x), up(np.asarray(tokens, np.uint32)), up(rng.random(16).astype(np.float32))
    for off in ([0, 5, 17, 17], [0xFFFFFFFF, 5, 16, 16], [9, 5, 5, 16]):
        path, counts, token = up(3 * 16 * 4), up(12), up(12)
        drafts.verify(device, b, t, up(np.array(off, np.uint32)), path, counts, token, parents=up(parents), accept=u, draws=u,
                      temperatures=u, sequences=3, rows=16, max_rows=16, vocab=500)
        c = device.read_array(counts, np.uint32, 3)
        n = [off[i + 1] - off[i] if 0 < off[i + 1] - off[i] <= 16 and off[i + 1] <= 16 else 0 for i in range(3)]
        assert [bool(v) for v in c] == [bool(v) for v in n]


# ---- kept rows ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("kv,d,page,layers", [(2, 64, 64, 3), (1, 64, 32, 1), (3, 128, 32, 2), (8, 128, 256, 1)])
@pytest.mark.parametrize("most", [1, 5, 16, 64])
def test_keep(device, up, kv, d, page, layers, most):  # noqa: F811
    rng = np.random.default_rng(kv + d + most)
    ns = [most, 1, max(1, most // 2), most, 0, most, most]
    lengths = [n + int(x) for n, x in zip(ns, [0, 40, 31, 57, 9, 64, 130])]
    width = max(-(-n // page) for n in lengths) + 1
    pages = sum(-(-n // page) for n in lengths) + 2
    table = tables(rng, lengths, page, pages, width)
    P = [Pages(pages, kv, d, page) for _ in range(layers)]
    for p in P:
        p.pool[:] = rng.integers(0, 256, p.pool.shape, dtype=np.uint8)
    pool = up(np.concatenate([p.pool for p in P], 1))
    path = np.full((len(ns), most), NO_ROW, np.uint32)
    counts = np.zeros(len(ns), np.uint32)
    for i, n in enumerate(ns):
        chosen = np.flatnonzero(rng.random(n) < 0.5)
        if i == 3:  # any order, rows again
            chosen = rng.integers(0, n, n)
        if i == 5:  # all of them: nothing moves
            chosen = np.arange(n)
        path[i, : len(chosen)] = chosen
        counts[i] = len(chosen)
    counts[6] = 0xFFFFFFFF  # past the rows: all, of which those that are none stay
    cache = kv4.Kv4Cache(device, kv, d, pages, page, layers=layers, pool=pool)
    new = up(np.full(len(ns) + 1, 5, np.uint32))
    cache.keep(up(path), up(counts), up(offsets_of(ns, 3)), up(np.array(lengths, np.uint32)), up(table), new, max_rows=most,
               sequences=len(ns), max_pages=width)
    for p in P:
        want = keep(p, table, path, counts, ns, lengths, page)
    got = device.read_array(new, np.uint32, len(ns) + 1)
    np.testing.assert_array_equal(got[:-1], want)
    assert got[-1] == 5
    np.testing.assert_array_equal(device.read_array(pool, np.uint8, pages * layers * P[0].bytes).reshape(pages, -1),
                                  np.concatenate([p.pool for p in P], 1))


def test_keep_what_does_not_fit(device, up):  # noqa: F811
    """Fewer positions than rows, more rows than max_rows, pages that are none, lengths past every table."""
    rng = np.random.default_rng(9)
    kv, d, page = 2, 64, 32
    P = Pages(6, kv, d, page)
    P.pool[:] = rng.integers(0, 256, P.pool.shape, dtype=np.uint8)
    pool = up(P.pool.copy())
    ns, lengths = [6, 9, 8, 8, 5, 3], [5, 60, 36, 36, 0xFFFFFFFF, 70]
    table = np.array([[0, 1], [2, 3], [4, NO_PAGE], [NO_PAGE, 5], [0, 1], [2, 3]], np.uint32)
    path = np.tile(np.array([0, 2, 3, 6, 7, 7, 7, 7], np.uint32), (6, 1))
    counts = np.array([3, 3, 5, 5, 3, 2], np.uint32)
    cache = kv4.Kv4Cache(device, kv, d, 6, page, pool=pool)
    new = up(4 * 6)
    cache.keep(up(path), up(counts), up(offsets_of(ns)), up(np.array(lengths, np.uint32)), up(table), new, max_rows=8, sequences=6,
               max_pages=2)
    want = keep(P, table, path, counts, ns, lengths, page)
    np.testing.assert_array_equal(device.read_array(new, np.uint32, 6), want)
    np.testing.assert_array_equal(device.read_array(pool, np.uint8, P.pool.size).reshape(P.pool.shape), P.pool)


# ---- refusals -----------------------------------------------------------------------------------------


def test_refusals(device, up):  # noqa: F811
    b = up(1 << 16)

    def fails(match, call, error=_lib.EgError):
        with pytest.raises(error, match=match):
            call()

    table = lambda **c: drafts.rope_table(device, b, **{**dict(positions=1, rotary_dim=64), **c})  # noqa: E731
    for r in (0, 12, 520):
        fails(f"rotary_dim {r}", lambda: table(rotary_dim=r))
    fails("theta 0", lambda: table(theta=0.0))
    fails("theta nan", lambda: table(theta=float("nan")))
    fails("factor -2", lambda: table(scaling="linear", factor=-2.0))
    fails("factor inf", lambda: table(scaling="base", factor=float("inf")))
    fails("context 0", lambda: table(scaling="turns"))
    fails("low 4, high 4", lambda: table(scaling="log_turns", context=8.0, low=4.0))
    fails("amplitude nan", lambda: table(amplitude=float("nan")))
    fails("under 2\\^31", lambda: table(first=2 ** 31, positions=1), _lib.EgRangeError)
    fails("16-byte aligned", lambda: drafts.rope_table(device, K.Binding(b, 8), positions=1, rotary_dim=64))
    fails("NULL argument", lambda: drafts.rope_table(device, None, positions=1, rotary_dim=64))
    table(positions=0)

    ok = dict(rows=2, head_dim=64, table_positions=4, q=b, q_out=b, heads=2, offsets=b, sequences=1)
    turn = lambda **c: drafts.rope(device, b, **{**ok, **c})  # noqa: E731
    fails("head_dim 60", lambda: turn(head_dim=60))
    fails("head_dim 520", lambda: turn(head_dim=520))
    fails("rotary_dim 72", lambda: turn(rotary_dim=72))
    fails("rotary_dim 12", lambda: turn(rotary_dim=12))
    fails("go together", lambda: turn(heads=0))
    fails("go together", lambda: turn(q_out=None))
    fails("go together", lambda: turn(kv_heads=1))
    fails("go together", lambda: turn(k=b, k_out=b))
    fails("starts and sequences go with offsets", lambda: turn(offsets=None))
    fails("starts and sequences go with offsets", lambda: turn(offsets=None, sequences=0, starts=b, positions=b))
    fails("NULL argument", lambda: turn(offsets=None, sequences=0))
    fails("strides 132", lambda: turn(q_stride=132, q_out_stride=132))
    fails("strides 128, 0, 64", lambda: turn(q_out_stride=64))
    fails("16-byte aligned", lambda: turn(q=K.Binding(b, 8)))
    fails("its type and stride", lambda: turn(out_type="f16"))
    fails("its type and stride", lambda: turn(q_stride=136))
    fails("rows over the grid limit", lambda: turn(rows=1 << 30), _lib.EgRangeError)
    fails("65536 and 0 heads", lambda: turn(heads=65536), _lib.EgRangeError)
    turn(rows=0, q=None, q_out=None, heads=0)
    turn(sequences=0)

    cache = kv4.Kv4Cache(device, 2, 64, 3, 64, pool=b)
    ok = dict(heads=2, rows=1, max_rows=1, sequences=1, max_pages=1)
    tree = lambda *a, **c: cache.attend_tree(*(a or (b, b, b, b, b)), **{**ok, **c})  # noqa: E731
    fails("heads 3 are not a multiple", lambda: tree(heads=3))
    fails("max_rows 65", lambda: tree(max_rows=65), _lib.EgRangeError)
    fails("scale -1", lambda: tree(scale=-1.0))
    fails("strides 132", lambda: tree(q_stride=132))
    fails("strides 128, 64", lambda: tree(out_stride=64))
    fails("16-byte aligned", lambda: tree(K.Binding(b, 4), b, b, b, b))
    for i in range(5):
        fails("NULL argument", lambda: tree(*[None if j == i else b for j in range(5)]))
    fails("over the grid limit", lambda: tree(rows=1 << 29), _lib.EgRangeError)
    fails("layer 1 of 1", lambda: tree(layer=1), _lib.EgRangeError)
    cache.dims.head_dim = 96
    fails("head_dim 96 is not supported", tree)
    cache.dims.head_dim = 64
    tree(None, None, None, None, None, rows=0)
    tree(None, None, None, None, None, max_rows=0)
    tree(None, None, None, None, None, sequences=0)

    ok = dict(sequences=1, rows=1, max_rows=1, vocab=8)
    check = lambda *a, **c: drafts.verify(device, *(a or (b,) * 6), **{**ok, **c})  # noqa: E731
    fails("max_rows 65", lambda: check(max_rows=65), _lib.EgRangeError)
    fails("vocab 0", lambda: check(vocab=0), _lib.EgRangeError)
    fails("vocab 1048577", lambda: check(vocab=(1 << 20) + 1), _lib.EgRangeError)
    fails("draft probabilities go with chains", lambda: check(draft=b, parents=b))
    fails("strides 7, 0", lambda: check(logits_stride=7))
    fails("strides 0, 7", lambda: check(draft_stride=7))
    for i in range(6):
        fails("NULL argument", lambda: check(*[None if j == i else b for j in range(6)]))
    fails("NULL argument", lambda: check(temperatures=b, draws=b))
    fails("NULL argument", lambda: check(temperatures=b, accept=b))
    fails("not aligned to their type", lambda: check(K.Binding(b, 2), b, b, b, b, b))
    fails("over the workspace or the grid limit", lambda: check(rows=65536), _lib.EgRangeError)
    fails("65536 sequences, 1 rows", lambda: check(sequences=1 << 16), _lib.EgRangeError)
    check(None, None, None, None, None, None, sequences=0)

    ok = dict(max_rows=1, sequences=1, max_pages=1)
    kept = lambda *a, **c: cache.keep(*(a or (b,) * 6), **{**ok, **c})  # noqa: E731
    fails("max_rows 65", lambda: kept(max_rows=65), _lib.EgRangeError)
    for i in range(6):
        fails("NULL argument", lambda: kept(*[None if j == i else b for j in range(6)]))
    cache.layers = 2
    fails("2 layers of 9216 bytes in pages of 9216", kept)
    cache.layers = 0
    fails("layer 0 of 0", kept, _lib.EgRangeError)
    cache.layers = 1
    kept(None, None, None, None, None, None, sequences=0)
    fails("out of range", lambda: kept(max_rows=-1), _lib.EgRangeError)
    assert _lib.load().eg_verify_drafts(device.ctx, *[None] * 12) == _lib.EG_ERR_INVALID
    assert _lib.load().eg_rope(device.ctx, *[None] * 9) == _lib.EG_ERR_INVALID
    bad = drafts._VERIFY_DIMS(1, 1, 1, 8, 0, 0, 3)
    assert _lib.load().eg_verify_drafts(device.ctx, *[ctypes.c_void_p(b.ptr)] * 11, bad) == _lib.EG_ERR_INVALID
    device.sync()


def test_outputs_that_lie_in_an_input_are_refused(device, up):  # noqa: F811
    """A sequence's workgroups read its inputs while its first one writes."""
    words = lambda n: up(np.zeros(n, np.uint32))  # noqa: E731
    cache = kv4.Kv4Cache(device, 1, 64, 2, 32)
    path, counts, offsets, lengths, table, new = words(12), words(3), words(4), words(3), words(3), words(3)
    keep_rows = lambda to: cache.keep(path, counts, offsets, lengths, table, to, max_rows=4, sequences=3, max_pages=1)  # noqa: E731
    for to in (lengths, counts, offsets, K.Binding(offsets, 12), path, K.Binding(path, 44), K.Binding(lengths, 8)):
        with pytest.raises(_lib.EgError, match="new_lengths lie in an input"):
            keep_rows(to)
    keep_rows(new)
    logits, ins = up(np.zeros((6, 8), np.float32)), dict(tokens=words(6), offsets=words(4), parents=words(6), accept=words(6), draws=words(3),
                                                        temperatures=words(3))
    outs = dict(path=words(12), counts=words(3), next=words(3))

    def check(**c):
        a = {**ins, **outs, **c}
        drafts.verify(device, logits, a["tokens"], a["offsets"], a["path"], a["counts"], a["next"], sequences=3, rows=6, max_rows=4, vocab=8,
                      parents=a["parents"], accept=a["accept"], draws=a["draws"], temperatures=a["temperatures"])

    for name in outs:
        for b in ins.values():
            with pytest.raises(_lib.EgError, match="an output lies in an input"):
                check(**{name: b})
    with pytest.raises(_lib.EgError, match="an output lies in an input"):
        check(next=K.Binding(ins["tokens"], 20))
    check()
    device.sync()
    cache.release()


# ---- together, captured, on other streams -------------------------------------------------------------


class Model:
    """Two layers of attention over the cache and a table of logits, in float64 from the definitions: what the step's
    launches are checked against. A token's rows are its embedding times fixed matrices."""

    heads, kv, d, layers, vocab = 6, 2, 64, 2, 97

    def __init__(self, rng):
        h = self.heads * self.d
        self.embedding = rng.standard_normal((self.vocab, 32)).astype(np.float32)
        self.wq, self.wk, self.wv = ([rng.standard_normal((32, n * self.d)).astype(np.float32) / 5 for _ in range(self.layers)]
                                     for n in (self.heads, self.kv, self.kv))
        self.wo = [rng.standard_normal((h, self.vocab)).astype(np.float32) / 4 for _ in range(self.layers)]


def speculate(device, up, rng, capture, temperature):  # noqa: F811
    """Steps of three sequences with trees of different sizes - rope, append, tree attention per layer, verify, keep -
    as a program runs them, each checked against float64 over the rows the reference keeps by itself."""
    M = Model(rng)
    heads, kv, d, layers, vocab, page, pages_n, width = M.heads, M.kv, M.d, M.layers, M.vocab, 32, 24, 6
    pages = kv4.PageTable(pages_n, page)
    cache = kv4.Kv4Cache(device, kv, d, pages_n, page, layers=layers)
    rope = up(256 * d * 4)
    drafts.rope_table(device, rope, positions=256, rotary_dim=d)
    cs = device.read_array(rope, np.float32, 256 * d).reshape(256, d // 2, 2)
    seqs, ns, most = [pages.create() for _ in range(3)], [7, 1, 4], 7
    total, off = sum(ns), offsets_of([7, 1, 4])
    rows_of = [[(np.zeros((0, kv, d)), np.zeros((0, kv, d))) for _ in range(layers)] for _ in seqs]
    dev = {n: up(4 * m) for n, m in dict(q=total * heads * d, k=total * kv * d, v=total * kv * d, qr=total * heads * d,
                                         kr=total * kv * d, start=3, length=3, table=3 * width, parents=total, depth=total,
                                         tokens=total, path=3 * most, counts=3, next=3, new=3, accept=total, draws=3, heat=3,
                                         logits=total * vocab, out=total * heads * d, off=4).items()}
    device.write(dev["off"], off)
    common = dict(sequences=3, max_pages=width)

    def layer(i):
        drafts.rope(device, rope, rows=total, head_dim=d, table_positions=256, q=dev["q"], q_out=dev["qr"], heads=heads, k=dev["k"],
                    k_out=dev["kr"], kv_heads=kv, positions=dev["depth"], offsets=dev["off"], starts=dev["start"], sequences=3)
        cache.append(dev["kr"], dev["v"], dev["off"], dev["start"], dev["table"], rows=total, layer=i, **common)
        cache.attend_tree(dev["qr"], dev["off"], dev["length"], dev["table"], dev["out"], parents=dev["parents"], heads=heads,
                          rows=total, max_rows=most, layer=i, **common)

    def finish():
        drafts.verify(device, dev["logits"], dev["tokens"], dev["off"], dev["path"], dev["counts"], dev["next"],
                      parents=dev["parents"], accept=dev["accept"], draws=dev["draws"], temperatures=dev["heat"], sequences=3,
                      rows=total, max_rows=most, vocab=vocab)
        cache.keep(dev["path"], dev["counts"], dev["off"], dev["length"], dev["table"], dev["new"], max_rows=most, **common)

    graphs = {}
    if capture:
        for name, what in [(i, lambda i=i: layer(i)) for i in range(layers)] + [("finish", finish)]:
            device.sync()
            device.capture_begin()
            what()
            graphs[name] = device.capture_end()
    run = lambda name: graphs[name].launch() if capture else (finish() if name == "finish" else layer(name))  # noqa: E731
    roots, emitted = [5, 50, 90], 0
    for step in range(6):
        parents = np.concatenate([random_tree(rng, n, 3) for n in ns])
        depth = np.concatenate([drafts.depths(parents[off[i]:off[i + 1]]) for i in range(3)])
        tokens = rng.integers(0, vocab, total).astype(np.uint32)
        tokens[off[:-1]] = roots
        starts = [pages.grow(s, n) for s, n in zip(seqs, ns)]
        lengths = [a + n for a, n in zip(starts, ns)]
        table = pages.table(seqs, width)
        accept, draws = rng.random(total).astype(np.float32), rng.random(3).astype(np.float32)
        heat = np.array([temperature, 0.0, temperature], np.float32)
        for n, x in dict(start=np.array(starts, np.uint32), length=np.array(lengths, np.uint32), table=table, parents=parents,
                         depth=depth, tokens=tokens, accept=accept, draws=draws, heat=heat).items():
            device.write(dev[n], x)
            device.sync()
        hidden = M.embedding[tokens]
        logits = np.zeros((total, vocab), np.float32)
        for i in range(layers):
            hq, hk, hv = ((hidden @ w[i]).reshape(total, -1, d) for w in (M.wq, M.wk, M.wv))
            for n, x in (("q", hq), ("k", hk), ("v", hv)):
                device.write(dev[n], x)
                device.sync()
            run(i)
            got = device.read_array(dev["out"], np.float32, hq.size).reshape(hq.shape)
            for s in range(3):
                r = slice(off[s], off[s + 1])
                at = starts[s] + depth[r].astype(int)
                qr, kr = rotate(hq[r], cs[at], d, "half"), rotate(hk[r], cs[at], d, "half")
                old = rows_of[s][i]
                new = tuple(np.concatenate([a[: starts[s]], held(b)]) for a, b in zip(old, (kr, hv[r])))
                rows_of[s][i] = new
                want, seen = tree_attend(qr.astype(np.float64), *new, 0.125, parents[r], np.ones(lengths[s], bool))
                for j in range(ns[s]):
                    bound = decode_bound(qr[j].astype(np.float64), *new, 0.125, seen[j], want[j], "f32")
                    assert np.all(np.abs(got[r][j] - want[j]) <= bound), (step, i, s, j)
            logits += got.reshape(total, -1) @ M.wo[i]
        # drafts that the model likes, so that branches are long: the parent's largest for the first child
        first = np.repeat(off[:-1], ns)
        for r in range(total):
            p = int(parents[r])
            if r != first[r] and rng.random() < 0.6:
                tokens[r] = int(logits[first[r] + p].argmax())
        logits *= 3.0
        device.write(dev["tokens"], tokens)
        device.write(dev["logits"], logits)
        device.sync()
        run("finish")
        path, counts, token = verify_all(logits, tokens, off, parents, None, accept, draws, heat, most)
        np.testing.assert_array_equal(device.read_array(dev["path"], np.uint32, 3 * most).reshape(3, most), path)
        np.testing.assert_array_equal(device.read_array(dev["counts"], np.uint32, 3), counts)
        np.testing.assert_array_equal(device.read_array(dev["next"], np.uint32, 3), token)
        np.testing.assert_array_equal(device.read_array(dev["new"], np.uint32, 3), np.array(starts) + counts)
        for s in range(3):
            kept = [starts[s] + int(j) for j in path[s, : counts[s]]]
            assert pages.shrink(seqs[s], ns[s] - int(counts[s])) == starts[s] + counts[s]
            for i in range(layers):
                rows_of[s][i] = tuple(np.concatenate([x[: starts[s]], x[kept]]) for x in rows_of[s][i])
                n = len(rows_of[s][i][0])
                ko, vo = up(4 * n * kv * d), up(4 * n * kv * d)
                cache.read(ko, vo, up(np.array([0, n], np.uint32)), up(np.zeros(1, np.uint32)), up(pages.table([seqs[s]], width)),
                           rows=n, sequences=1, max_pages=width, layer=i, out_type="f32")
                for o, x in zip((ko, vo), rows_of[s][i]):
                    np.testing.assert_array_equal(device.read_array(o, np.float32, x.size).reshape(x.shape), x)
            emitted += int(counts[s])
        roots = token.tolist()
    assert emitted > 18  # (drafts were accepted)
    for g in graphs.values():
        g.destroy()
    device.sync()
    cache.release()


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_speculative_run(device, up, temperature):  # noqa: F811
    speculate(device, up, np.random.default_rng(31), False, temperature)


def test_speculative_run_captured(device, up):  # noqa: F811
    speculate(device, up, np.random.default_rng(32), True, 1.0)


def test_two_captured_graphs_share_the_workspace(device, up):  # noqa: F811
    """A split tree attention and a verification, each captured: launched in turn, with eager calls between."""
    rng = np.random.default_rng(33)
    heads, kv, d, page, n, length, vocab = 4, 1, 64, 64, 12, 3000, 9000
    P, _, _ = random_pages(rng, 50, kv, d, page)
    cache = kv4.Kv4Cache(device, kv, d, 50, page, pool=up(P.pool))
    bq, tb = up(rng.standard_normal((n, heads, d)).astype(np.float32)), up(rng.permutation(50).astype(np.uint32)[None])
    off, ln = up(np.array([0, n], np.uint32)), up(np.array([length], np.uint32))
    x, tokens, _, q = verify_case(rng, [n], vocab, True, True)
    bx, bt, bd, u = up(x), up(tokens.astype(np.uint32)), up(q), up((np.full(n, 0.9999)).astype(np.float32))
    heat, draws = up(np.ones(1, np.float32)), up(np.full(1, 0.5, np.float32))
    outs = [(up(n * heads * d * 4), up(n * 4), up(4), up(4)) for _ in range(2)]

    def attend(o):
        cache.attend_tree(bq, off, ln, tb, o[0], heads=heads, rows=n, max_rows=n, sequences=1, max_pages=50)

    def check(o):
        drafts.verify(device, bx, bt, off, o[1], o[2], o[3], draft=bd, accept=u, draws=draws, temperatures=heat, sequences=1, rows=n,
                      max_rows=n, vocab=vocab)

    read = lambda o: [device.read_array(b, np.uint32, m).tolist() for b, m in zip(o, (n * heads * d, n, 1, 1))]  # noqa: E731
    attend(outs[0])
    check(outs[0])
    want = read(outs[0])
    device.sync()
    graphs = []
    for what in (attend, check):
        device.capture_begin()
        what(outs[1])
        graphs.append(device.capture_end())
    for turn in range(4):
        for b, m in zip(outs[1], (n * heads * d, n, 1, 1)):
            device.zero(b, 4 * m)
        for g in graphs if turn % 2 else graphs[::-1]:
            g.launch()
            (check if turn % 2 else attend)(outs[0])
        assert read(outs[1]) == want and read(outs[0]) == want
    for g in graphs:
        g.destroy()


def test_on_a_callers_stream(device, up):  # noqa: F811
    """Launches go to the stream that the context is given (another context's here), after what is on it."""
    rng = np.random.default_rng(34)
    owner = K.Device(0)
    dev = K.Device(0, stream=owner.stream)
    x, tokens, parents, _ = verify_case(rng, [9, 5], 151936, False, False)
    off, want = np.array([0, 9, 14], np.uint32), None
    b, t, p, o = up(np.zeros_like(x)), up(tokens.astype(np.uint32)), up(parents), up(off)
    outs = [(up(18 * 4), up(8), up(8)) for _ in range(2)]
    device.sync()
    owner.write(b, x)  # (on the stream, before the launch that reads it)
    drafts.verify(dev, b, t, o, *outs[0], parents=p, sequences=2, rows=14, max_rows=9, vocab=151936)
    owner.zero(b, x.nbytes)
    want = verify_all(x, tokens, off, parents, None, None, None, None, 9)
    for buf, w in zip(outs[0], want):
        np.testing.assert_array_equal(dev.read_array(buf, np.uint32, w.size).reshape(w.shape), w)
    dev.sync()
    dev.close()
    owner.close()
