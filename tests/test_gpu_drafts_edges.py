"""The operators of a speculative step at the ends of their ranges. The definitions (drafts_reference.py) are test_gpu_drafts.py's."""

import numpy as np
import pytest

from drafts_reference import NO_ROW, verify
from enargeia_amd import _lib, drafts, kv4
from enargeia_amd import kernels as K
from kv4_reference import as_type, random_pages
from test_gpu_drafts import check_verify, random_tree, verify_case
from test_gpu_kv4 import kv4_size, offsets_of, up  # noqa: F401 (a fixture)

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
