"""The speculative step without a GPU: the page table's bookkeeping, the trees' depths, names and ranges, and that
the definition of the verification (drafts_reference.py) leaves the target's distribution as it is."""

import ctypes
import os
import re

import numpy as np
import pytest

from drafts_reference import frequencies, keep, rotate, sees, verify
from enargeia_amd import _lib, drafts, kv4
from kv4_reference import random_pages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class NoDevice:
    ctx = None


def test_sequences_shrink_and_grow_again():
    t = kv4.PageTable(8, 32)
    a = t.create()
    assert t.grow(a, 70) == 0 and len(t.held[a]) == 3
    assert t.shrink(a, 0) == 70 and len(t.held[a]) == 3
    assert t.shrink(a, 6) == 64 and len(t.held[a]) == 2 and t.free_pages == 6
    assert t.grow(a, 1) == 64 and t.length[a] == 65
    assert t.shrink(a, np.uint32(65)) == 0 and t.held[a] == [] and t.free_pages == 8
    with pytest.raises(_lib.EgRangeError, match="cannot shrink by 1 rows"):
        t.shrink(a, 1)
    with pytest.raises(_lib.EgRangeError, match="cannot shrink by -1 rows"):
        t.shrink(a, -1)


def test_a_page_that_a_fork_shares_is_not_shrunk_into():
    t = kv4.PageTable(8, 32)
    a = t.create()
    t.grow(a, 64)
    b = t.fork(a)  # both pages shared, nothing to copy
    t.grow(a, 3)
    assert t.shrink(a, 3) == 64  # (its own third page)
    with pytest.raises(_lib.EgError, match="a fork shares that page"):
        t.shrink(a, 1)
    assert t.length[a] == 64 and len(t.held[a]) == 2
    assert t.shrink(a, 32) == 32  # whole pages: the next rows lie in a new one
    assert t.users[t.held[b][1]] == 1
    t.free(b)
    assert t.shrink(a, 1) == 31


def test_shrinking_leaves_what_a_fork_has_still_to_copy():
    t = kv4.PageTable(4, 32)
    a = t.create()
    t.grow(a, 40)
    b = t.fork(a)
    source = t.held[a][1]
    assert t.copies == [(source, t.held[b][1])]
    t.shrink(a, 40)
    assert source not in t._free() and t.copies == [(source, t.held[b][1])]
    t.shrink(b, 8)  # (the copy's target is free again: nobody reads it)
    assert t.copies == []


def test_depths():
    np.testing.assert_array_equal(drafts.depths([-1, 0, 1, 0, 3, 3, 2]), [0, 1, 2, 1, 2, 2, 3])
    np.testing.assert_array_equal(drafts.depths(np.array([0xFFFFFFFF, 0, 1, 9, 3], np.uint32)), [0, 1, 2, 0, 1])
    assert drafts.depths([]).dtype == np.uint32


def test_names_and_ranges():
    text = open(os.path.join(ROOT, "include", "enargeia_hip.h")).read()
    values = dict((n, int(v)) for n, v in re.findall(r"(EG_ROPE_\w+) = (\d)", text))
    assert drafts.SCALINGS == {n[8:].lower() if n != "EG_ROPE_PLAIN" else "none": v for n, v in values.items()
                               if n not in ("EG_ROPE_HALF", "EG_ROPE_INTERLEAVED")}
    assert drafts.LAYOUTS == {"half": values["EG_ROPE_HALF"], "interleaved": values["EG_ROPE_INTERLEAVED"]}
    with pytest.raises(_lib.EgError, match="scaling 'yes'"):
        drafts.rope_table(NoDevice, 0, positions=1, rotary_dim=64, scaling="yes")
    with pytest.raises(_lib.EgError, match="layout 'both'"):
        drafts.rope(NoDevice, 0, rows=1, head_dim=64, table_positions=1, layout="both")
    with pytest.raises(_lib.EgError, match="element type 'q4'"):
        drafts.verify(NoDevice, 0, 0, 0, 0, 0, 0, sequences=1, rows=1, max_rows=1, vocab=8, type="q4")
    with pytest.raises(_lib.EgRangeError, match="out of range"):
        drafts.verify(NoDevice, 0, 0, 0, 0, 0, 0, sequences=1 << 32, rows=1, max_rows=1, vocab=8)
    with pytest.raises(_lib.EgRangeError, match="out of range"):
        drafts.rope(NoDevice, 0, rows=-1, head_dim=64, table_positions=1)
    with pytest.raises(_lib.EgRangeError, match="out of range"):
        drafts.rope_table(NoDevice, 0, positions=1, first=1 << 32, rotary_dim=64)
    for call in (lambda: drafts.rope_table(NoDevice, 0, positions=1, rotary_dim=64),
                 lambda: drafts.rope(NoDevice, 0, rows=1, head_dim=64, table_positions=1),
                 lambda: drafts.verify(NoDevice, 0, 0, 0, 0, 0, 0, sequences=1, rows=1, max_rows=1, vocab=8)):
        with pytest.raises(_lib.EgError, match="ctx is NULL"):
            call()
    lib = _lib.load()
    assert lib.eg_attention_tree_kv4(*[None] * 10) == _lib.EG_ERR_INVALID
    assert lib.eg_kv4_keep_rows(*[None] * 9, 1, 1) == _lib.EG_ERR_INVALID


def test_dims_are_laid_out_as_the_header_has_them():
    text = open(os.path.join(ROOT, "include", "enargeia_hip.h")).read()
    size = {"uint32_t": 4, "int": 4, "float": 4, "double": 8, "uint64_t": 8}

    def packed(name):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1), flags=re.S)
        at = 0
        for kind, names in re.findall(r"(\w+)\s+([\w\s,]+);", body):
            for _ in names.split(","):
                at = -(-at // size[kind]) * size[kind] + size[kind]
        return at

    assert packed("eg_rope_table_dims") == len(drafts._TABLE_DIMS(*[0] * 10))
    assert packed("eg_rope_dims") == len(drafts._ROPE_DIMS(*[0] * 14))
    assert packed("eg_verify_dims") == len(drafts._VERIFY_DIMS(*[0] * 7))
    assert packed("eg_attention_tree_dims") == len(kv4._ATTENTION_TREE_DIMS(*[0] * 6, 0.0))


# ---- the definitions ----------------------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotations_add_up(layout):
    """Rotated by m and then by n is rotated by m + n; lengths stay."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 3, 24)).astype(np.float32)
    f = frequencies(16, 1e4)
    cs = lambda p: np.stack([np.cos(p * f), np.sin(p * f)], -1)[None].astype(np.float32)  # noqa: E731
    once, twice = rotate(x, cs(12), 16, layout), rotate(rotate(x, cs(5), 16, layout), cs(7), 16, layout)
    np.testing.assert_allclose(once, twice, atol=32 * 2.0 ** -24)  # (a dozen roundings of values under 4)
    np.testing.assert_allclose((once.astype(np.float64) ** 2).sum(-1), (x.astype(np.float64) ** 2).sum(-1), rtol=1e-6)
    np.testing.assert_array_equal(once[..., 16:], x[..., 16:])


def test_scaled_frequencies():
    f = frequencies(64, 1e4)
    np.testing.assert_allclose(frequencies(64, 1e4, "linear", 4.0), f / 4)
    base = frequencies(64, 1e4, "base", 4.0)
    np.testing.assert_allclose([base[0], base[-1]], [f[0], f[-1] / 4])  # the shortest wave stays, the longest is stretched
    for s in ("turns", "log_turns"):
        g = frequencies(64, 1e4, s, 4.0, 2048.0, 1.0, 8.0)
        turns = 2048 * f / (2 * np.pi)
        np.testing.assert_allclose(g[turns >= 8], f[turns >= 8])
        np.testing.assert_allclose(g[turns <= 1], f[turns <= 1] / 4)
        assert np.all(np.diff(g) < 0)


def softmax(x):
    e = np.exp(x - x.max())
    return e / e.sum()


def test_a_drawn_draft_leaves_the_targets_distribution():
    """Over all drafts (each as likely as q draws it) and a grid of the two random numbers, the token after the root
    is distributed as p; each of `grid` steps of a number is off by one step at most where an id's border lies."""
    rng = np.random.default_rng(2)
    vocab, grid = 5, 100
    x = rng.standard_normal((2, vocab)) * 1.5
    q = softmax(rng.standard_normal(vocab)).astype(np.float32)
    draft = np.stack([q, q])
    u = (np.arange(grid) + 0.5) / grid
    got = np.zeros(vocab)
    for y in range(vocab):
        for a in u:
            path, token = verify(x, [0, y], None, draft, [0, a], 0.5, 0.8)
            if len(path) == 2:
                got[y] += q[y] / grid
                continue
            for d in u:
                got[verify(x, [0, y], None, draft, [0, a], d, 0.8)[1]] += q[y] / grid / grid
    assert np.all(np.abs(got - softmax(x[0] / 0.8)) <= (vocab + 1) / grid)


def test_chosen_drafts_leave_the_targets_distribution():
    rng = np.random.default_rng(3)
    vocab, grid = 5, 40
    x = rng.standard_normal((4, vocab)) * 1.5
    tokens, parents = [0, 3, 1, 3], [-1, 0, 0, 0]  # (the third holds the first's token again)
    u = (np.arange(grid) + 0.5) / grid
    got = np.zeros(vocab)
    for a in u:
        for b in u:
            path, _ = verify(x, tokens, parents, None, [0, a, b, 0.0], 0.5, 1.0)
            if len(path) == 2:
                assert path[1] != 3
                got[tokens[path[1]]] += 1 / grid ** 2
            else:
                for d in u:
                    t = verify(x, tokens, parents, None, [0, a, b, 0.0], d, 1.0)[1]
                    assert t not in (3, 1)
                    got[t] += 1 / grid ** 3
    assert np.all(np.abs(got - softmax(x[0])) <= 3.0 / grid)


def test_greedy_takes_the_branch_of_the_largest_logits():
    x = np.zeros((5, 6))
    x[0, [2, 4]] = 3.0  # (2: the lowest of equals)
    x[1, 5], x[3, 1] = 1.0, 1.0
    tokens, parents = [0, 4, 9, 2, 1], [-1, 0, 0, 0, 3]
    assert verify(x, tokens, parents, None, None, 0, 0.0) == ([0, 3, 4], 0)
    assert verify(x, [0, 4, 2, 3, 1], parents, None, None, 0, 0.0) == ([0, 2], 0)


def test_who_sees_whom():
    m = sees([-1, 0, 0, 2, 9, 4], 6)
    want = [[0], [0, 1], [0, 2], [0, 2, 3], [4], [4, 5]]
    assert [list(np.flatnonzero(r)) for r in m] == want
    np.testing.assert_array_equal(sees(None, 4), np.tril(np.ones((4, 4), bool)))


def test_reference_keeps_rows():
    rng = np.random.default_rng(4)
    P, k, v = random_pages(rng, 3, 2, 64, 32)
    table = np.array([[2, 0]], np.uint32)
    before = P.pool.copy()
    new = keep(P, table, np.array([[0, 2, 5, 0xFFFFFFFF, 0, 0]], np.uint32), [3], [6], [36], 32)
    assert new.tolist() == [33]
    where = lambda p: (table[0][p // 32], p % 32)  # noqa: E731
    for i, j in ((0, 0), (1, 2), (2, 5), (3, 3), (5, 5)):
        kk, vv = P.get(*where(30 + i), 1)
        np.testing.assert_array_equal(kk, k[where(30 + j)][1])
        np.testing.assert_array_equal(vv, v[where(30 + j)][1])
    np.testing.assert_array_equal(P.pool[1], before[1])


def test_library_has_the_entry_points():
    lib = _lib.load()
    for name in ("eg_rope_table", "eg_rope", "eg_attention_tree_kv4", "eg_verify_drafts", "eg_kv4_keep_rows"):
        assert isinstance(getattr(lib, name), ctypes._CFuncPtr)
