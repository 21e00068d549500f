"""The 4-bit cache's format and the host's bookkeeping of its pages, without a GPU."""

import numpy as np
import pytest

from enargeia_amd import kv4
from enargeia_amd._lib import EgError, EgRangeError
from enargeia_amd.kernels import Buffer
from kv4_reference import Pages, by_the_text, halfway, held, quantize, random_pages, scale_of


def test_page_bytes():
    assert kv4.page_bytes(2, 64, 64) == 2 * 64 * 72
    assert kv4.page_bytes(8, 128, 256) == 8 * 256 * 144


def test_values_are_exact_in_f16_and_within_half_a_step():
    rng = np.random.default_rng(1)
    for spread in (1e-6, 1e-3, 1.0, 300.0, 6e4):
        x = np.asarray(rng.standard_normal((500, 64)) * spread, np.float32)
        y = held(x)
        assert np.array_equal(y, y.astype(np.float16).astype(np.float64))
        s = scale_of(np.abs(x.reshape(500, 2, 32)).max(-1)).astype(np.float64)
        off = np.abs(y - x).reshape(500, 2, 32)
        # a code is at most half a step off, and one clamped at 7 by what the scale was rounded down:
        # half a step of 8 significant bits (2^-8) of absmax = 7 steps, within half a step
        # (values over 65408 saturate)
        inside = np.abs(x).reshape(500, 2, 32) <= 65408
        assert np.all((off <= 0.5001 * s[..., None] + 2.0 ** -19)[inside])


def test_not_finite_groups_are_nan():
    x = np.ones((1, 64), np.float32)
    x[0, 3] = np.inf
    assert np.isnan(held(x)[0, :32]).all() and np.array_equal(held(x)[0, 32:], held(np.ones((1, 64), np.float32))[0, 32:])


def test_reference_places_what_it_reads():
    rng = np.random.default_rng(2)
    for d, page in ((64, 32), (128, 64)):
        P, k, v = random_pages(rng, 3, 2, d, page)
        Q = Pages(3, 2, d, page, fill=0xA5)
        for p in range(3):
            for slot in range(page):
                for h in range(2):
                    got = P.get(p, slot, h)
                    assert np.array_equal(got[0], k[p, slot, h]) and np.array_equal(got[1], v[p, slot, h])
                    Q.put(p, slot, h, k[p, slot, h], v[p, slot, h])
        c, _ = quantize(np.asarray(k, np.float32))
        assert c.min() >= 1 and c.max() <= 15
        for p, slot, h in ((0, 0, 0), (2, page - 1, 1), (1, 13, 0)):
            assert np.array_equal(Q.get(p, slot, h)[0], held(np.asarray(k[p, slot, h], np.float32)))


def test_pages_grow_fork_free_compact():
    t = kv4.PageTable(8, 32)
    a = t.create()
    assert t.grow(a, 40) == 0 and t.held[a] == [0, 1] and t.free_pages == 6
    b = t.fork(a)  # one whole page shared, the partial one copied
    assert t.held[b] == [0, 2] and t.users[:3] == [2, 1, 1]
    c = t.fork(b)  # the copy is still pending: from where its rows come
    assert t.copies == [(1, 2), (1, 3)] and t.users[0] == 3
    t.free(a)
    assert t.users[:4] == [2, 0, 1, 1]
    d = t.create()
    t.grow(d, 1)
    assert t.held[d] == [4]  # not page 1: it is still to be copied from
    assert np.array_equal(t.take_copies(), np.array([[1, 2], [1, 3]], np.uint32)) and t.copies == []
    assert t.grow(b, 60) == 40 and t.held[b] == [0, 2, 1, 5]
    t.free(d)
    t.free(b)
    assert t.compact() == 2 and t.held[c] == [0, 1]
    assert np.array_equal(t.take_copies(), np.array([[3, 1]], np.uint32))
    assert t.free_pages == 6 and t.users[:3] == [1, 1, 0]
    assert np.array_equal(t.table([c], 3), np.array([[0, 1, kv4.NO_PAGE]], np.uint32))
    assert t.lengths([c])[0] == 40


def test_whole_pages_fork_without_a_copy():
    t = kv4.PageTable(4, 32)
    a = t.create()
    t.grow(a, 64)
    b = t.fork(a)
    assert t.held[b] == t.held[a] and t.copies == []
    t.grow(a, 1)
    t.grow(b, 1)
    assert t.held[a][2] != t.held[b][2]


def test_page_table_refusals():
    t = kv4.PageTable(2, 32)
    a = t.create()
    with pytest.raises(EgRangeError, match="3 pages wanted, 2 of 2 free"):
        t.grow(a, 65)
    assert t.lengths([a])[0] == 0 and t.held[a] == [] and t.free_pages == 2
    t.grow(a, 33)
    with pytest.raises(EgRangeError, match="1 pages wanted, 0 of 2 free"):
        t.fork(a)
    assert t.users == [1, 1]
    with pytest.raises(EgRangeError, match="has 2 pages, the table 1"):
        t.table([a], 1)
    with pytest.raises(EgError, match="page_size 48"):
        kv4.PageTable(2, 48)
    t.free(a)
    b = t.create()
    t.grow(b, 3)
    t.fork(b)
    with pytest.raises(EgError, match="copies of forks are pending"):
        t.compact()


def test_element_types_have_names():
    with pytest.raises(EgError, match="element type 'f8'"):
        kv4.attention_packed(None, 0, 0, 0, 0, 0, 0, sequences=1, rows=1, key_rows=1, heads=1, kv_heads=1,
                             head_dim=64, type="f8")


def test_dimensions_out_of_range():
    class Device:
        ctx = None

    with pytest.raises(EgRangeError, match="a dimension out of range"):
        kv4.attention_packed(Device, 0, 0, 0, 0, 0, 0, sequences=-1, rows=1, key_rows=1, heads=1, kv_heads=1, head_dim=64)
    cache = kv4.Kv4Cache(Device, 1, 64, 4, 32, pool=1 << 20)
    with pytest.raises(EgRangeError, match="a dimension out of range"):
        cache.attend(0, 0, 0, 0, heads=1 << 32, sequences=1, max_pages=1)
    with pytest.raises(EgRangeError, match="layer 1 of 1"):
        cache.read(0, 0, 0, 0, 0, rows=1, sequences=1, max_pages=1, layer=1)


def test_pools_too_small_or_released():
    class Device:
        ctx = None

        def buffer(self, size, label=""):
            return Buffer(self, 1 << 20, size, label)

    size = 4 * kv4.page_bytes(1, 64, 32) * 2
    with pytest.raises(EgRangeError, match=f"a pool of {size - 1} bytes for 4 pages of {size // 4}"):
        kv4.Kv4Cache(Device(), 1, 64, 4, 32, layers=2, pool=Buffer(Device(), 1 << 20, size - 1))
    with pytest.raises(EgRangeError, match="a pool of"):
        kv4.Kv4Cache(Device(), 1, 64, 4, 32, layers=2, pool=np.zeros(size - 1, np.uint8))
    with pytest.raises(EgRangeError, match="a pool of 0 pages of 2 layers"):
        kv4.Kv4Cache(Device(), 1, 64, 0, 32, layers=2)
    pool = Buffer(Device(), 1 << 20, size)
    cache = kv4.Kv4Cache(Device(), 1, 64, 4, 32, layers=2, pool=pool)
    pool.ptr = 0  # released by its owner
    for call in (lambda: cache.read(0, 0, 0, 0, 0, rows=1, sequences=1, max_pages=1, layer=1),
                 lambda: cache.append(0, 0, 0, 0, 0, rows=1, sequences=1, max_pages=1, layer=1),
                 lambda: cache.attend(0, 0, 0, 0, heads=1, sequences=1, max_pages=1, layer=1)):
        with pytest.raises(EgError, match="the pool has been released"):
            call()
    owner = kv4.Kv4Cache(Device(), 1, 64, 4, 32, layers=2)
    owner.owned.ptr = 0  # (nothing of a device to free)
    owner.release()
    with pytest.raises(EgError, match="the pool has been released"):
        owner.read(0, 0, 0, 0, 0, rows=1, sequences=1, max_pages=1, layer=1)


def test_sizes_past_32_bits_are_refused():
    """Not taken modulo 2^32, which is a call that returns with nothing done."""
    class Device:
        ctx = None

    cache = kv4.Kv4Cache(Device, 1, 64, 4, 32, pool=1 << 20)
    some = dict(rows=1, sequences=1, max_pages=1)
    calls = [lambda **c: cache.read(0, 0, 0, 0, 0, **{**some, **c}), lambda **c: cache.append(0, 0, 0, 0, 0, **{**some, **c})]
    for name in some:
        for size in (1 << 32, (1 << 32) + 1, -1):
            for call in calls:
                with pytest.raises(EgRangeError, match="a dimension out of range"):
                    call(**{name: size})
    for name in ("sequences", "max_pages"):
        with pytest.raises(EgRangeError, match=f"a dimension out of range .{name} 4294967296"):
            cache.attend(0, 0, 0, 0, **{"heads": 1, "sequences": 1, "max_pages": 1, name: 1 << 32})
    for count in (1 << 32, -1):
        with pytest.raises(EgRangeError, match="a dimension out of range"):
            cache.copy_pages(0, count)
    # (the largest that fit are the library's to check)
    with pytest.raises(EgError, match="ctx is NULL"):
        cache.read(0, 0, 0, 0, 0, rows=(1 << 32) - 1, sequences=(1 << 32) - 1, max_pages=(1 << 32) - 1)


def test_pools_past_64_bits_are_refused():
    class Device:
        ctx = None

    for change in (dict(kv_heads=(1 << 32) + 1), dict(head_dim=(1 << 32) + 64), dict(page_size=(1 << 32) + 32)):
        with pytest.raises(EgRangeError, match="a dimension out of range"):
            kv4.page_bytes(**{"kv_heads": 1, "head_dim": 64, "page_size": 32, **change})
    size = kv4.page_bytes(1, 64, 32)
    with pytest.raises(EgRangeError, match="pages 4294967300"):
        kv4.Kv4Cache(Device, 1, 64, (1 << 32) + 4, 32, pool=1 << 20)
    with pytest.raises(EgRangeError, match="pool_bytes"):  # (its stride modulo 2^64 is one layer's)
        kv4.Kv4Cache(Device, 1, 64, 4, 32, layers=(1 << 64) // 256 + 1, pool=np.zeros(4 * size, np.uint8))


def test_sequences_do_not_shrink():
    """Grown by fewer than no rows, a sequence kept its pages, and a fork of it shared one that both then wrote."""
    t = kv4.PageTable(8, 32)
    a = t.create()
    t.grow(a, 64)
    with pytest.raises(EgRangeError, match="cannot grow by -40 rows"):
        t.grow(a, -40)
    assert t.length[a] == 64 and t.held[a] == [0, 1] and t.grow(a, 0) == 64
    b = t.fork(a)
    t.grow(a, 1)
    t.grow(b, 1)
    assert t.held[a] == [0, 1, 2] and t.held[b] == [0, 1, 3]


def test_free_pages_are_those_that_can_be_taken():
    t = kv4.PageTable(3, 32)
    a = t.create()
    t.grow(a, 40)
    t.fork(a)
    t.free(a)  # its second page is free, but still to be copied from
    c = t.create()
    assert t.free_pages == 0
    with pytest.raises(EgRangeError, match="1 pages wanted, 0 of 3 free"):
        t.grow(c, 1)
    t.take_copies()
    assert t.free_pages == 1
    t.grow(c, 1)
    assert t.held[c] == [1] and t.free_pages == 0


def test_formats_that_no_call_takes_have_no_size():
    class Device:
        ctx = None

        def buffer(self, size, label=""):
            raise AssertionError("a pool of an unknown format was allocated")

    for match, change in (("head_dim 96 is not supported", dict(head_dim=96)), ("page_size 48 is not supported", dict(page_size=48)),
                          ("0 kv heads", dict(kv_heads=0)), ("1025 kv heads", dict(kv_heads=1025))):
        dims = {"kv_heads": 2, "head_dim": 64, "page_size": 32, **change}
        with pytest.raises(EgError, match=match):
            kv4.page_bytes(**dims)
        with pytest.raises(EgError, match=match):
            kv4.Kv4Cache(Device(), pages=4, **dims)
    assert kv4.page_bytes(1024, 128, 256) == 1024 * 256 * 144


def test_scales_and_codes_by_the_headers_words():
    """The arithmetic that the header states, in exact rationals: values halfway between two codes, values of
    each type, the smallest and the largest scales."""
    rng = np.random.default_rng(3)
    ties, divided = halfway(rng)
    groups = [ties]
    for spread in (2.0 ** -20, 2.0 ** -18, 1e-3, 1.0, 300.0, 3e4, 1e9):
        x = np.asarray(rng.standard_normal((60, 32)) * spread, np.float32)
        with np.errstate(over="ignore"):
            h = x.astype(np.float16).astype(np.float32)
        groups += [x, h[np.isfinite(h).all(1)], (x.view(np.uint32) & 0xFFFF0000).view(np.float32)]
    x = np.concatenate(groups)
    codes, scales = quantize(x)
    for row, c, s in zip(x, codes, scales[:, 0].astype(np.float64)):
        want, scale = by_the_text(row)
        assert s == scale and c.tolist() == want
    # a value over its scale is another format: about one scale in four has ties that fall to the odd code
    other = (codes[: len(ties)] != divided).any(1).mean()
    assert 0.1 < other < 0.5, other


def test_pool_sizes_of_numpy_integers_do_not_wrap():
    """A pool that is allocated for pages counted in 32 bits holds all of them."""
    sizes = []

    class Device:
        ctx = None

        def buffer(self, size, label=""):
            sizes.append(size)
            return Buffer(self, 1 << 20, size, label)

    stride = kv4.page_bytes(8, 128, 64)
    cache = kv4.Kv4Cache(Device(), 8, 128, np.int32(60000), 64, layers=np.int32(1))
    kv4.Kv4Cache(Device(), 8, 128, 60000, 64, layers=np.int32(60000))
    assert sizes == [60000 * stride, 60000 * 60000 * stride] and cache.dims.pages == 60000
    large = kv4.Kv4Cache(Device(), 1024, 128, 4, 256, layers=64)
    assert large._at(np.int32(63)) == (1 << 20) + 63 * kv4.page_bytes(1024, 128, 256)


@pytest.mark.parametrize("kind", [np.uint32, np.int32, np.uint64, np.uint8])
def test_sequences_grow_by_numpy_integers(kind):
    """As `lengths` gives them."""
    t = kv4.PageTable(12, 32)
    a = t.create()
    assert t.grow(a, kind(200)) == 0 and len(t.held[a]) == 7
    assert t.grow(a, kind(100)) == 200 and len(t.held[a]) == 10 and t.length[a] == 300
    b = t.create()
    t.grow(b, t.lengths([b])[0])
    assert t.held[b] == [] and t.lengths([a, b]).tolist() == [300, 0]
