"""The operators over the paged 4-bit cache in the forms that only large or uneven calls take, against the
same float64 references and bounds as tests/test_gpu_kv4.py: codes read past the caches (a reach over 256
MiB), more steps than a wave holds page ids for, appends and reads of more than 2048 rows. And scales and
codes by the header's words."""

import numpy as np
import pytest

from enargeia_amd import kv4
from kv4_reference import NO_PAGE, as_type, attend, by_the_text, from_type, halfway, random_pages
from test_gpu_kv4 import check_append, check_decode, decode_bound, kv4_size, up  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_scales_and_codes_by_the_headers_words(device, up, kind):  # noqa: F811
    """Values halfway between two codes, of every scale's significand."""
    ties, divided = halfway(np.random.default_rng(3))
    d, page = 64, 64
    x = ties.reshape(-1, d)
    n = len(x)
    raw, values = as_type(x, kind)
    pages = -(-n // page)
    cache = kv4.Kv4Cache(device, 1, d, pages, page, pool=up(pages * kv4.page_bytes(1, d, page)))
    off, st, tb = up(np.array([0, n], np.uint32)), up(np.zeros(1, np.uint32)), up(np.arange(pages, dtype=np.uint32)[None])
    b, k, v = up(raw), up(n * d * 4), up(n * d * 4)
    cache.append(b, b, off, st, tb, rows=n, sequences=1, max_pages=pages, in_type=kind)
    cache.read(k, v, off, st, tb, rows=n, sequences=1, max_pages=pages, out_type="f32")
    want, by_division = [], []
    for group, other in zip(values.reshape(-1, 32), divided):
        codes, scale = by_the_text(group)
        want.append((np.array(codes) - 8.0) * scale)
        by_division.append((other - 8.0) * scale)
    assert kind != "f32" or np.any(np.stack(want) != np.stack(by_division))
    for o in (k, v):
        np.testing.assert_array_equal(device.read_array(o, np.float32, n * d).reshape(-1, 32), np.stack(want))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,page", [(14, 2, 64, 64), (12, 1, 64, 64), (32, 8, 128, 64), (16, 1, 128, 128)])
def test_decode_tables_that_reach_past_256_mib(device, up, heads, kv, d, page, kind):  # noqa: F811
    """Tables and a pool that reach over the Infinity Cache's size, of which a few pages anywhere are named."""
    print(f"decode of a large pool, {heads}/{kv} x {d}, page {page}, {kind}", flush=True)
    rng = np.random.default_rng(heads + d)
    size = kv4.page_bytes(kv, d, page)
    pages = (1 << 28) // size + 5
    lengths = [1300, 0, 65]
    width = -(-pages // len(lengths))
    assert min(len(lengths) * width, pages) * size > 1 << 28
    need = [-(-n // page) for n in lengths]
    P, kv_k, kv_v = random_pages(rng, sum(need), kv, d, page)
    at = rng.choice(pages - 1, sum(need), replace=False)
    at[0] = pages - 1
    table = np.full((len(lengths), width), NO_PAGE, np.uint32)
    mine, first = [], 0  # the sequences' pages among those of P
    for i, c in enumerate(need):
        mine.append(np.arange(first, first + c))
        table[i, :c] = at[mine[i]]
        first += c
        if lengths[i] % page:  # past the sequence's end: nothing to be attended to
            for h in range(kv):
                _, _, ks, vs = P._streams(mine[i][-1], h)
                ks[:, lengths[i] % page:] = np.nan
                vs[:, lengths[i] % page:] = np.inf
    pool = up(pages * size)
    for i, p in enumerate(at):
        device.write(pool, P.pool[i], offset=int(p) * size)
    device.sync()
    q = rng.standard_normal((len(lengths), heads, d)).astype(np.float32)
    raw, val = as_type(q, kind)
    out = up(q.size * kv4_size(kind))
    kv4.Kv4Cache(device, kv, d, pages, page, pool=pool).attend(
        up(raw), up(np.array(lengths, np.uint32)), up(table), out, heads=heads, sequences=len(lengths), max_pages=width,
        type=kind)
    got = from_type(device.read(out, q.size * kv4_size(kind)), kind).reshape(q.shape)
    for i, n in enumerate(lengths):
        k, v = (x[mine[i]].reshape(-1, kv, d)[:n] for x in (kv_k, kv_v))
        seen = np.ones(n, bool)
        want = attend(val[i], k, v, d ** -0.5, seen)
        off, bound = np.abs(got[i] - want), decode_bound(val[i], k, v, d ** -0.5, seen, want, kind)
        assert np.all(off <= bound), f"sequence {i} of {n}: off by {np.max(off / bound):.2f} of the bound"


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,d,page", [(5, 64, 64), (4, 128, 64), (5, 64, 32), (9, 128, 128)])
def test_decode_more_steps_than_a_wave_holds_page_ids(device, up, heads, d, page, kind):  # noqa: F811
    """So many sequences that none is split: a wave then goes through more than the 64 steps whose page ids
    it holds at a time - just those, one more, and a ragged end."""
    whole = 64 * 4 * (64 if heads <= 8 and page >= 64 else 32)  # steps x waves x positions of a step
    lengths = [0] * 600
    lengths[::40] = [1] * 15
    lengths[3], lengths[200], lengths[599] = whole, whole + 1, whole + 777
    print(f"decode of {whole} positions and more, {heads}/1 x {d}, page {page}, {kind}", flush=True)
    check_decode(device, up, np.random.default_rng(page + d), lengths, heads, 1, d, page, kind)


@pytest.mark.parametrize("heads,kv,d,page,in_type,out_type", [
    (2, 1, 128, 64, "f32", "bf16"), (10, 1, 128, 32, "bf16", "f32"), (5, 2, 64, 256, "bf16", "f32"), (33, 1, 64, 32, "f32", "f16")])
def test_append_and_read_more_than_2048_rows(device, up, heads, kv, d, page, in_type, out_type):  # noqa: F811
    """Whole blocks a wave, queries of several rows a workgroup, from positions inside the blocks of 8 and of 32."""
    print(f"append of 2300 rows, {heads}/{kv} x {d}, page {page}, {in_type} to {out_type}", flush=True)
    check_append(device, up, np.random.default_rng(heads), [1500, 3, 0, 797], [3, 8, 40, 29], heads, kv, d, page, in_type,
                 out_type, before=5, after=2)
