"""The operators of a speculative step at the ends of their ranges: sizes past a workgroup's first turn of each loop, offsets that
do not ascend, temperatures next to f32's largest, scores past 2^20, memory behind the outputs, and outputs that overlap. The definitions
(drafts_reference.py) and their bounds are test_gpu_drafts.py's."""

import numpy as np
import pytest

from drafts_reference import NO_ROW, keep, tree_attend, verify, verify_all
from enargeia_amd import _lib, drafts, kv4
from enargeia_amd import kernels as K
from kv4_reference import Pages, as_type, from_type, random_pages
from test_gpu_drafts import check_rope, check_tree, check_verify, random_tree, verify_case
from test_gpu_kv4 import decode_bound, kv4_size, offsets_of, tables, up  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


# ---- verification -------------------------------------------------------------------------------------


def run_verify(device, up, logits, tokens, off, parents, accept, draws, temperatures, max_rows):  # noqa: F811
    s, (rows, vocab) = len(off) - 1, logits.shape
    path, counts, token = up(np.full((s, max_rows), 5, np.uint32)), up(np.full(s, 5, np.uint32)), up(np.full(s, 5, np.uint32))
    f32 = lambda a: None if a is None else up(np.asarray(a, np.float32))  # noqa: E731
    drafts.verify(device, up(logits), up(np.asarray(tokens, np.uint32)), up(np.array(off, np.uint32)), path, counts, token,
                  parents=up(parents), accept=f32(accept), draws=f32(draws), temperatures=f32(temperatures), sequences=s, rows=rows,
                  max_rows=max_rows, vocab=vocab)
    return (device.read_array(path, np.uint32, s * max_rows).reshape(s, max_rows), device.read_array(counts, np.uint32, s),
            device.read_array(token, np.uint32, s))


@pytest.mark.parametrize("hot", [False, True])
@pytest.mark.parametrize("off", [[9, 5, 5, 16], [0xFFFFFFFF, 5, 16, 16], [0, 5, 17, 17], [8, 12, 0, 6], [12, 16, 4, 12, 0, 4]])
def test_verify_of_offsets_that_do_not_ascend(device, up, off, hot):  # noqa: F811
    """What a sequence that is computed is given comes from this call's logits, wherever the others lie."""
    for seed in range(4):
        rng = np.random.default_rng(10 * seed + hot)
        rows, vocab, s = 16, 9000, len(off) - 1
        before, tokens, _, _ = verify_case(rng, [rows], vocab, False, False)
        logits, tokens, _, _ = verify_case(rng, [rows], vocab, False, False)
        parents = np.full(rows, NO_ROW, np.uint32)
        want = np.full((s, rows), NO_ROW, np.uint32), np.zeros(s, np.uint32), np.full(s, NO_ROW, np.uint32)
        accept, draws = rng.random(rows), rng.random(s)
        heat = rng.uniform(0.5, 1.5, s) if hot else None
        f32 = np.float32
        for i in range(s):
            a, b = off[i], off[i + 1]
            if not 0 < b - a <= rows or b > rows:
                continue
            parents[a:b] = random_tree(rng, b - a, 2)
            for r in range(a + 1, b):  # drafts that are often accepted
                if rng.random() < 0.7:
                    tokens[r] = logits[a + int(parents[r])].argmax()
            got, want[2][i] = verify(logits[a:b], tokens[a:b], parents[a:b], None, f32(accept[a:b]), f32(draws[i]),
                                     f32(heat[i]) if hot else 0.0)
            want[1][i] = len(got)
            want[0][i, : len(got)] = got
        run_verify(device, up, before, tokens, [0, rows], parents, accept, draws[:1], heat[:1] if hot else None, rows)
        for x, y, name in zip(run_verify(device, up, logits, tokens, off, parents, accept, draws, heat, rows), want, ("path", "counts", "next")):
            np.testing.assert_array_equal(x, y, err_msg=name)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("temperature", [2.0 ** 120, 2.0 ** 121, 1e37, 1e38, 3.4e38])
def test_verify_temperatures_next_to_the_largest(device, up, temperature, kind):  # noqa: F811
    """Logits of both signs next to f32's largest: their differences pass it, and at such a temperature still count."""
    vocab, rows = 5000, 4
    for top, rest in ((3.38e38, -3.38e38), (3.38e38, -np.inf), (3.38e38, 0.0)):
        x = np.full((rows, vocab), rest, np.float32)
        x[:, 3:9] = (np.linspace(0.9, 1.0, 6) * top).astype(np.float32)
        x[:, 4100:4105] = -top
        x[:, 20] = 1.0
        for accept in (0.004, 0.02, 0.1, 0.3, 0.6):
            for draw in (0.05, 0.95):
                check_verify(device, up, x, [0, 8, 7, 4102], [rows], None, None, np.full(rows, accept), [draw], [temperature], kind)
                check_verify(device, up, x, [0, 8, 20, 4102], [rows], np.array([9, 0, 0, 0], np.uint32), None, np.full(rows, accept), [draw],
                             [temperature], kind)
        q = np.full((rows, vocab), 1.0 / vocab, np.float32)
        check_verify(device, up, x, [0, 8, 7, 4102], [rows], None, q, np.full(rows, 0.9), [0.4], [temperature], kind)


@pytest.mark.parametrize("how", ["chain", "tree", "draft"])
@pytest.mark.parametrize("chunks,seqs", [(7, 620), (11, 760)])
def test_verify_of_more_chunks_than_a_workgroup_takes_at_once(device, up, chunks, seqs, how):  # noqa: F811
    """More than 16 and 32 chunks a CU: a workgroup draws from 8 and 12, four at a time, the last of them partial."""
    rng = np.random.default_rng(chunks + len(how))
    vocab = 4096 * chunks - 700
    ns = [1 + (i % 7 == 3) for i in range(seqs)]
    x, tokens, parents, draft = verify_case(rng, ns, vocab, how != "tree", how == "draft")
    t = np.where(rng.random(seqs) < 0.95, rng.uniform(0.5, 1.5, seqs), 0.0)
    check_verify(device, up, x, tokens, ns, parents, draft, rng.random(sum(ns)), rng.random(seqs), t)


@pytest.mark.parametrize("hot", [False, True])
def test_verify_writes_its_outputs_alone(device, up, hot):  # noqa: F811
    """Words behind path, counts and next stay, whether sequences are computed or not."""
    rng = np.random.default_rng(43)
    ns, width = [5, 0, 9, 2, 1], 5
    x, tokens, parents, _ = verify_case(rng, ns, 5000, False, False)
    s, rows, off = len(ns), sum(ns), offsets_of(ns)
    sizes = (s * width, s, s)
    outs = [up(np.full(n + 80, 0xA5A5A5A5, np.uint32)) for n in sizes]
    accept, draws, heat = (rng.random(n).astype(np.float32) for n in (rows, s, s))
    heat = heat + np.float32(0.5) if hot else None
    drafts.verify(device, up(x), up(np.asarray(tokens, np.uint32)), up(off), *outs, parents=up(parents), accept=up(accept), draws=up(draws),
                  temperatures=up(heat) if hot else None, sequences=s, rows=rows, max_rows=width, vocab=5000)
    want = verify_all(x, tokens, off, parents, None, accept, draws, heat, width)
    for b, n, w in zip(outs, sizes, want):
        got = device.read_array(b, np.uint32, n + 80)
        np.testing.assert_array_equal(got[:n].reshape(w.shape), w)
        assert np.all(got[n:] == 0xA5A5A5A5)


def test_verify_rows_that_the_workspace_does_not_hold_are_refused(device, up):  # noqa: F811
    b = up(64)
    check = lambda **c: drafts.verify(device, *[b] * 6, **{**dict(sequences=1, rows=16383, max_rows=1, vocab=1 << 20), **c})  # noqa: E731
    for c in (dict(), dict(vocab=(1 << 20) - 4095), dict(rows=16382, accept=b, draws=b, temperatures=b), dict(sequences=65536, vocab=8),
              dict(rows=65536, vocab=8)):
        with pytest.raises(_lib.EgRangeError, match="over the workspace or the grid limit"):
            check(**c)


# ---- rotary positions and kept rows -------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv,rotary", [(32, 8, 128), (32, 8, 64), (40, 8, 128), (40, 8, 64), (40, 8, 40)])
def test_rope_of_rows_longer_than_a_workgroups_turn(device, up, layout, heads, kv, rotary):  # noqa: F811
    rng = np.random.default_rng(heads + rotary)
    for kinds in (("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f32", "f16")):
        check_rope(device, up, rng, [3, 0, 6], [7, 9, 30], None, heads, kv, 128, rotary, layout, *kinds, before=1, after=2)
        if kinds[0] == kinds[1]:
            check_rope(device, up, rng, [5], [11], None, heads, kv, 128, rotary, layout, *kinds, in_place=True, pad=8)


@pytest.mark.parametrize("kv,d,layers,seqs", [(5, 64, 33, 110), (4, 128, 64, 100)])
def test_keep_of_several_heads_a_wave(device, up, kv, d, layers, seqs):  # noqa: F811
    """More (layer, kv head, sequence) than waves the device holds: two and three of a wave's, which do not divide them."""
    rng = np.random.default_rng(kv)
    page, most = 32, 4
    ns = [int(n) for n in rng.integers(1, most + 1, seqs)]
    lengths = [n + int(x) for n, x in zip(ns, rng.integers(0, 40, seqs))]
    width = max(-(-n // page) for n in lengths)
    pages = sum(-(-n // page) for n in lengths)
    table = tables(rng, lengths, page, pages, width)
    P = [Pages(pages, kv, d, page) for _ in range(layers)]
    for p in P:
        p.pool[:] = rng.integers(0, 256, p.pool.shape, dtype=np.uint8)
    pool = up(np.concatenate([p.pool for p in P], 1))
    path, counts = np.full((seqs, most), NO_ROW, np.uint32), np.zeros(seqs, np.uint32)
    for i, n in enumerate(ns):
        chosen = np.flatnonzero(rng.random(n) < 0.6)
        path[i, : len(chosen)], counts[i] = chosen, len(chosen)
    cache = kv4.Kv4Cache(device, kv, d, pages, page, layers=layers, pool=pool)
    new = up(4 * seqs)
    cache.keep(up(path), up(counts), up(offsets_of(ns)), up(np.array(lengths, np.uint32)), up(table), new, max_rows=most, sequences=seqs,
               max_pages=width)
    for p in P:
        want = keep(p, table, path, counts, ns, lengths, page)
    np.testing.assert_array_equal(device.read_array(new, np.uint32, seqs), want)
    np.testing.assert_array_equal(device.read_array(pool, np.uint8, pages * layers * P[0].bytes).reshape(pages, -1),
                                  np.concatenate([p.pool for p in P], 1))


# ---- the tree attention -------------------------------------------------------------------------------


def far_scores(rng, pages, kv, d, page):
    """A pool whose keys are 4 in dim 0, a whole number from -7 to 7 in dim 32 and 0 elsewhere; keys and values."""
    P, _, v = random_pages(rng, pages, kv, d, page)
    k = np.zeros((pages, page, kv, d))
    k[..., 0], k[..., 32] = 4, rng.integers(-7, 8, (pages, page, kv))
    for p in range(pages):
        for h in range(kv):
            kw, _, ks, _ = P._streams(p, h)
            ks[:] = 1
            kw[:] = 0x88888888
            kw[:, 0, 0] = 0x8888888C
            kw[:, 0, 1] = 0x88888880 + (k[p, :, h, 32] + 8).astype(np.uint32)
    return P, k, v


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv,ns,most", [(4, 1, [5, 1], 32), (4, 2, [16, 9], 300), (64, 8, [8] * 36, 200), (64, 8, [16] * 36, 200),
                                              (64, 8, [40] * 36, 130), (64, 8, [32] * 32, 200)])
def test_tree_of_scores_past_2_to_20(device, up, heads, kv, ns, most, d, kind):  # noqa: F811
    """Scores of +-2^20 and half numbers up to 3.5 beside them, in heads between ordinary ones: what the largest part adds to all of a
    head's is the same, so the outputs are those of queries without it. Every product and sum of a score is exact (23 bits at most), and
    so is a score less the largest one; what is left is the ordinary bound of the rest. Where a head's positions meet by the waves'
    maxima in f32 (few columns, more than a wave's 32 positions) each of the two maxima, of 1.5 x 2^20 in powers of two, is rounded by up
    to 2^-4, so shares of the weights are off by factors from 2^(-1/8) to 2^(1/8), and an output by up to 2^(1/4) - 1 of the largest value. Weights of 16-bit rows are scaled by 2^12 at least, of which half a step of
    f16's smallest numbers is 2^-37."""
    rng = np.random.default_rng(len(ns) * most + d)
    page, seqs, group = 32, len(ns), heads // kv
    lengths = [max(n, most - 7 * (i % 9)) for i, n in enumerate(ns)]
    width = -(-max(lengths) // page) + 12
    pages = max(-(-n // page) for n in lengths)
    P, kk, vv = far_scores(rng, pages, kv, d, page)
    order = rng.permutation(pages).astype(np.uint32)
    table = np.full((seqs, width), 0xFFFFFFFF, np.uint32)
    table[:, :pages] = order
    kk, vv = (x[order].reshape(-1, kv, d) for x in (kk, vv))
    parents = np.concatenate([random_tree(rng, n) for n in ns])
    q = np.zeros((sum(ns), heads, d), np.float32)
    q[..., 32] = 2.0 ** -4
    far = np.arange(sum(ns))[:, None] + np.arange(heads) * 3
    q[..., 0] = np.array([0.0, 2.0 ** 15, -2.0 ** 15], np.float32)[far % 3]
    raw, val = as_type(q, kind)
    np.testing.assert_array_equal(val, q)
    out = up(raw.nbytes)
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(P.pool))
    cache.attend_tree(up(raw), up(offsets_of(ns)), up(np.array(lengths, np.uint32)), up(table), out, parents=up(parents), heads=heads,
                      rows=sum(ns), max_rows=max(ns), sequences=seqs, max_pages=width, type=kind, scale=8.0)
    got = from_type(device.read(out, raw.nbytes), kind).reshape(q.shape)
    meet = 2.0 ** 0.25 - 1 if max(ns) * group <= 64 and most > 32 else 0.0
    off = offsets_of(ns)
    near = val.copy()
    near[..., 0] = 0.0
    for s in range(0, seqs, 5):
        r = slice(int(off[s]), int(off[s + 1]))
        k, v = kk[: lengths[s]], vv[: lengths[s]]
        want, seen = tree_attend(val[r], k, v, 8.0, parents[r], np.ones(lengths[s], bool))
        for j in range(ns[s]):
            bound = decode_bound(near[r][j], k, v, 8.0, seen[j], want[j], kind)
            bound = bound + (seen[j].sum() * 2.0 ** -37 + meet) * np.abs(v).max() + (2.0 ** -25 if kind == "f16" else 0.0)
            off_by = np.abs(got[r][j] - want[j])
            assert np.all(off_by <= bound), (s, j, float(np.nanmax(off_by / bound)))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,d,page,n,length,seqs", [(32, 8, 128, 256, 32, 256, 32), (32, 8, 128, 256, 13, 200, 33), (64, 8, 64, 256, 32, 255, 32),
                                                           (64, 8, 64, 32, 16, 32, 36), (64, 8, 64, 32, 32, 64, 32), (14, 2, 64, 128, 16, 128, 16),
                                                           (8, 8, 128, 256, 1, 512, 40), (4, 1, 64, 32, 3, 3, 1)])
def test_tree_of_tables_as_wide_as_the_sequences(device, up, heads, kv, d, page, n, length, seqs, kind):  # noqa: F811
    """Tables of one page and of two, with no entry to spare. 16-bit rows' weights are scaled by 2^12 at least, of which half a step
    of f16's smallest numbers, 2^-25, is 2^-37."""
    rng = np.random.default_rng(page + n)
    ns = [n if i % 3 == 0 else int(rng.integers(1, n + 1)) for i in range(seqs)]
    lengths = [length if i % 3 == 0 else int(rng.integers(max(k, length // 3), length + 1)) for i, k in enumerate(ns)]
    check_tree(device, up, rng, ns, lengths, heads, kv, d, page, kind, extra=-1, floor=0.0 if kind == "f32" else 2.0 ** -37, step=4)


# ---- outputs that overlap -----------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_verify_outputs_in_the_logits_the_draft_or_each_other_are_refused(device, up, kind):  # noqa: F811
    """To the first and last word of them; what lies between their rows, or next to them, is no part of them."""
    rows, vocab, stride, size = 4, 10, 16, kv4_size(kind)
    logits, draft = up(np.zeros((rows, stride * size), np.uint8)), up(np.zeros((rows, stride), np.float32))
    words = lambda n: up(np.zeros(n, np.uint32))  # noqa: E731
    tokens, offsets, numbers, b = words(rows), up(np.array([0, 2, 4], np.uint32)), up(np.zeros(rows, np.float32)), words(64)

    def check(path=0, counts=64, token=128):
        a = [x if not isinstance(x, int) else K.Binding(b, x) for x in (path, counts, token)]
        drafts.verify(device, logits, tokens, offsets, *a, draft=draft, accept=numbers, draws=numbers, temperatures=numbers,
                      sequences=2, rows=rows, max_rows=3, vocab=vocab, type=kind, logits_stride=stride, draft_stride=stride)

    row, end = stride * size, vocab * size
    for at in (0, row + end - 4, 3 * row + end - 4):
        for name in ("path", "counts", "token"):
            with pytest.raises(_lib.EgError, match="an output lies in an input"):
                check(**{name: K.Binding(logits, at)})
    for at in (0, stride * 4 + 36, 3 * stride * 4 + 36):
        for name in ("path", "counts", "token"):
            with pytest.raises(_lib.EgError, match="an output lies in an input"):
                check(**{name: K.Binding(draft, at)})
    check(token=K.Binding(draft, 40), counts=K.Binding(logits, row + end))
    check(path=K.Binding(draft, 40))  # (24 bytes: the whole of what lies between two rows)
    for at in (dict(counts=0), dict(counts=20), dict(token=64), dict(token=68), dict(token=60), dict(path=44, counts=64), dict(path=108, token=128)):
        with pytest.raises(_lib.EgError, match="an output lies in another"):
            check(**at)
    check(path=0, counts=24, token=32)
    check(path=16, counts=0, token=8)
    device.sync()


def test_keep_of_lengths_in_the_table_or_the_pool_is_refused(device, up):  # noqa: F811
    """A new length written over a page id would send another workgroup's rows to a wrong page."""
    words = lambda n: up(np.zeros(n, np.uint32))  # noqa: E731
    kv, d, page, pages, layers, seqs = 1, 64, 32, 3, 2, 3
    size = kv4.page_bytes(kv, d, page) * layers
    pool, table = up(np.zeros(pages * (size + 64), np.uint8)), up(np.zeros((seqs, 2), np.uint32))
    cache = kv4.Kv4Cache(device, kv, d, pages, page, layers=layers, pool=pool)
    cache.dims.page_stride = size + 64  # (64 bytes of no page behind each)
    ok = dict(path=words(12), counts=words(seqs), offsets=words(seqs + 1), lengths=words(seqs), table=table, new=words(seqs))

    def kept(**c):
        a = {**ok, **c}
        cache.keep(a["path"], a["counts"], a["offsets"], a["lengths"], a["table"], a["new"], max_rows=4, sequences=seqs, max_pages=2)

    for at in (0, 20):
        with pytest.raises(_lib.EgError, match="new_lengths lie in an input"):
            kept(new=K.Binding(table, at))
    for at in (0, size - 4, size + 64, 3 * (size + 64) - 68):
        with pytest.raises(_lib.EgError, match="new_lengths lie in the pool"):
            kept(new=K.Binding(pool, at))
        for name in ("path", "counts", "offsets", "lengths", "table"):
            with pytest.raises(_lib.EgError, match="an input lies in the pool"):
                kept(**{name: K.Binding(pool, at)})
    kept(new=K.Binding(pool, size), lengths=K.Binding(pool, 2 * size + 64))  # (between pages)
    kept()
    device.sync()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_outputs_that_overlap_are_refused(device, up, layout):  # noqa: F811
    """An output that is its input, or lies between the rows of others, is taken; any other overlap is a race of workgroups."""
    rows, heads, kv, d = 5, 3, 2, 64
    wide = (heads + 2 * kv) * d  # q, k and v side by side
    b, far = up(np.zeros((rows + 3, wide), np.float32)), up(np.zeros((rows + 3, wide), np.float32))
    table, words = up(np.zeros((8, d), np.float32)), up(np.zeros(64, np.uint32))
    at = lambda row, head=0, of=b: K.Binding(of, (row * wide + head * d) * 4)  # noqa: E731
    ok = dict(rows=rows, head_dim=d, table_positions=8, q=at(0), heads=heads, k=at(0, heads), kv_heads=kv, positions=K.Binding(words, 0),
              offsets=K.Binding(words, 32), starts=K.Binding(words, 48), sequences=2, layout=layout, q_stride=wide, k_stride=wide,
              q_out_stride=wide, k_out_stride=wide)

    def turn(q_out, k_out, **c):
        drafts.rope(device, table, **{**ok, "q_out": q_out, "k_out": k_out, **c})

    turn(at(0), at(0, heads))  # in place
    turn(at(0, 0, far), at(0, heads, far))
    turn(at(0), at(0, heads + kv))  # k's rows over v's
    for q_out, k_out in ((at(1), at(0, heads)), (at(0, 1), at(0, 5)), (at(0, heads + kv), at(0, heads)), (at(0, 0, far), at(0, heads - 1)),
                         (at(0, 0, far), at(0, heads + 1)), (at(0, 0, far), at(2, heads)), (at(0, heads), at(0, 0, far)),
                         (at(0, 0, far), at(0)), (table, at(0, 0, far))):
        with pytest.raises(_lib.EgError, match="an output lies in an input"):
            turn(q_out, k_out)
    for offset, where in ((0, "positions"), (16, "positions"), (32, "offsets"), (48, "starts")):
        assert where in ok
        with pytest.raises(_lib.EgError, match="an output lies in an input"):
            turn(at(0, 0, far), K.Binding(words, offset))
    for k_out in (at(0, 2, far), at(0, 0, far), at(rows - 1, 1, far), at(1, 0, far)):
        with pytest.raises(_lib.EgError, match="q_out and k_out overlap"):
            turn(at(0, 0, far), k_out)
    with pytest.raises(_lib.EgError, match="an output lies in an input"):  # rows of another step
        turn(at(1), at(0, heads, far), q_out_stride=heads * d)
    turn(at(rows), at(0, heads, far), q_out_stride=heads * d)  # behind the rows of q and k
    device.sync()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,ns,lengths", [(4, 1, [5, 3], [40, 31]), (4, 1, [9], [3000]), (64, 8, [16] * 36, [90] * 36), (64, 8, [32] * 32, [140] * 32),
                                                 (64, 8, [8] * 36, [70] * 36)])
def test_tree_in_place(device, up, heads, kv, ns, lengths, kind):  # noqa: F811
    """The result in q's place, gaps between rows among it: the bits that it has elsewhere."""
    rng = np.random.default_rng(heads + len(ns))
    d, page, pad, seqs, rows = 64, 32, 16, len(ns), sum(ns)
    pages = -(-max(lengths) // page)
    P, _, _ = random_pages(rng, pages, kv, d, page)
    table = np.tile(rng.permutation(pages).astype(np.uint32), (seqs, 1))
    raw, _ = as_type(rng.standard_normal((rows, heads * d + pad)).astype(np.float32), kind)
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(P.pool))
    q, own = up(raw), up(raw)
    ins = [up(x) for x in (offsets_of(ns), np.array(lengths, np.uint32), table)]
    for out in (own, q):
        cache.attend_tree(q, *ins, out, parents=up(np.concatenate([random_tree(np.random.default_rng(n), n) for n in ns])), heads=heads, rows=rows,
                          max_rows=max(ns), sequences=seqs, max_pages=pages, type=kind, q_stride=heads * d + pad, out_stride=heads * d + pad)
    a, b = (device.read_array(x, np.uint8, raw.nbytes) for x in (own, q))
    np.testing.assert_array_equal(a, b)


def test_tree_results_that_lie_in_an_input_are_refused(device, up):  # noqa: F811
    kv, d, page, pages, heads, rows = 1, 64, 32, 3, 2, 6
    size = kv4.page_bytes(kv, d, page)
    cache = kv4.Kv4Cache(device, kv, d, pages, page, pool=up(pages * size))
    b, words = up(np.zeros((2 * rows + 1, heads * d), np.float32)), up(np.zeros(64, np.uint32))
    row = 4 * heads * d
    ins = [K.Binding(words, 64 * i) for i in range(4)]  # offsets, lengths, table, parents

    def attend(out, **c):
        cache.attend_tree(b, *ins[:3], out, parents=ins[3], **{**dict(heads=heads, rows=rows, max_rows=6, sequences=2, max_pages=2), **c})

    for out in (K.Binding(b, row), K.Binding(b, 16), K.Binding(b, 5 * row), *ins, cache.pool, K.Binding(cache.pool, pages * size - 16)):
        with pytest.raises(_lib.EgError, match="out lies in an input"):
            attend(out)
    with pytest.raises(_lib.EgError, match="out lies in an input"):  # of another step
        attend(b, out_stride=heads * d + 8)
    attend(b)
    attend(K.Binding(b, 6 * row))
    device.sync()
    cache.release()
