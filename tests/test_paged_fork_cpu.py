"""Sequences of a paged cache that go on from one another, and pools made dense again: the bookkeeping, on the host alone."""
import ctypes as C

import numpy as np
import pytest


@pytest.fixture
def cache(pkg):
    made = []

    def make(blocks=12, sequences=5, size=4):
        made.append(pkg.lib.cml_paged_kv_cache_create_device(blocks, sequences, size))
        return made[-1]
    yield make
    for c in made:
        pkg.lib.cml_paged_kv_cache_free(c)


def ids(c, s):
    t = c.contents.sequences[s]
    return [t.block_ids[i] for i in range(t.num_blocks)]


def fork(pkg, c, s):
    a, b = C.c_int(), C.c_int()
    return pkg.lib.cml_paged_cache_fork(c, s, a, b), a.value, b.value


@pytest.mark.parametrize("tokens", [0, 1, 3, 4, 5, 8, 11])
def test_a_fork_shares_full_blocks(pkg, cache, tokens):
    L, c = pkg.lib, cache()
    s = L.cml_paged_cache_init_sequence(c)
    assert L.cml_paged_cache_extend(c, s, tokens) == 0
    mine, free = ids(c, s), c.contents.free_count
    child, a, b = fork(pkg, c, s)
    full = tokens // 4
    assert child >= 0 and child != s and c.contents.sequences[child].seq_len == tokens
    assert ids(c, s) == mine and ids(c, child)[:full] == mine[:full]
    if tokens % 4:
        assert (a, b) == (mine[full], ids(c, child)[full]) and b not in mine and c.contents.free_count == free - 1
    else:
        assert (a, b) == (-1, -1) and ids(c, child) == mine and c.contents.free_count == free
    # each goes on by itself
    assert L.cml_paged_cache_extend(c, s, 6) == 0 and L.cml_paged_cache_extend(c, child, 9) == 0
    assert not set(ids(c, s)[full:]) & set(ids(c, child)[full:])
    L.cml_paged_cache_free_sequence(c, s)
    assert all(c.contents.blocks[i].in_use for i in ids(c, child))
    L.cml_paged_cache_free_sequence(c, child)
    assert c.contents.free_count == c.contents.num_blocks
    assert sorted(c.contents.free_list[i] for i in range(12)) == list(range(12))


def test_forks_of_forks_and_blocks_let_go(pkg, cache):
    L, c = pkg.lib, cache(16, 5, 4)
    s = L.cml_paged_cache_init_sequence(c)
    assert L.cml_paged_cache_extend(c, s, 21) == 0                       # five full, one begun
    x = fork(pkg, c, s)[0]
    y = fork(pkg, c, x)[0]
    assert c.contents.free_count == 8
    L.cml_paged_cache_release_before(c, s, 9)                             # two blocks of one sequence: the others still hold them
    assert c.contents.free_count == 8 and ids(c, s)[:2] == [-1, -1] and -1 not in ids(c, x)
    z, a, b = fork(pkg, c, s)                                             # from a sequence that let go of some
    assert ids(c, z)[:2] == [-1, -1] and ids(c, z)[2:5] == ids(c, s)[2:5] and c.contents.free_count == 7
    L.cml_paged_cache_free_sequence(c, x)
    L.cml_paged_cache_free_sequence(c, y)
    assert c.contents.free_count == 11                                    # their two begun blocks, and the two let go of first
    L.cml_paged_cache_free_sequence(c, s)
    assert c.contents.free_count == 12
    L.cml_paged_cache_free_sequence(c, z)
    assert c.contents.free_count == 16 and c.contents.num_sequences == 0


def test_fork_refusals(pkg, cache):
    L, c = pkg.lib, cache(3, 2, 4)
    a, b = C.c_int(), C.c_int()
    assert L.cml_paged_cache_fork(None, 0, a, b) == -1 and L.cml_paged_cache_fork(c, 0, a, b) == -1 and L.cml_paged_cache_fork(c, 9, a, b) == -1
    s = L.cml_paged_cache_init_sequence(c)
    assert L.cml_paged_cache_extend(c, s, 9) == 0
    assert fork(pkg, c, s) == (-1, -1, -1) and c.contents.num_sequences == 1          # no block for the begun one
    L.cml_paged_cache_free_sequence(c, s)
    s = L.cml_paged_cache_init_sequence(c)
    assert L.cml_paged_cache_extend(c, s, 5) == 0
    assert L.cml_paged_cache_fork(c, s, None, None) == -1                              # nowhere to say what to copy
    t = fork(pkg, c, s)[0]
    assert t >= 0 and c.contents.free_count == 0
    L.cml_paged_cache_free_sequence(c, t)
    assert L.cml_paged_cache_init_sequence(c) == t
    assert fork(pkg, c, s) == (-1, -1, -1) and c.contents.free_count == 1              # no slot; nothing was taken
    other = cache(2, 2, 4)
    s = L.cml_paged_cache_init_sequence(other)
    assert L.cml_paged_cache_extend(other, s, 8) == 0
    assert L.cml_paged_cache_fork(other, s, None, None) >= 0                           # nothing to copy


def test_compact(pkg, cache):
    L, c = pkg.lib, cache(24, 5, 4)
    seqs = [L.cml_paged_cache_init_sequence(c) for _ in range(4)]
    for n in (7, 5, 4, 9):
        for i, s in enumerate(seqs):
            assert L.cml_paged_cache_extend(c, s, 1 if n == 9 and i else min(n, 5)) == 0
    child = fork(pkg, c, seqs[3])[0]
    L.cml_paged_cache_free_sequence(c, seqs[0])
    L.cml_paged_cache_free_sequence(c, seqs[2])
    live = [seqs[1], seqs[3], child]
    was = {s: ids(c, s) for s in live}
    used = {i for s in live for i in was[s]}
    moves = np.full(2 * 24, -7, np.int32)
    n = L.cml_paged_cache_compact(c, pkg.np_ptr(moves))
    k = len(used)
    assert n == len([i for i in used if i >= k]) > 0 and (moves[2 * n:] == -7).all()
    m = dict(moves[:2 * n].reshape(-1, 2).tolist())
    assert set(m) == {i for i in used if i >= k} and set(m.values()) == set(range(k)) - used
    for s in live:
        assert ids(c, s) == [m.get(i, i) for i in was[s]]
    assert [c.contents.blocks[i].in_use for i in range(24)] == [i < k for i in range(24)]
    assert c.contents.free_count == 24 - k and sorted(c.contents.free_list[i] for i in range(24 - k)) == list(range(k, 24))
    assert L.cml_paged_cache_compact(c, pkg.np_ptr(moves)) == 0                        # nothing left to move
    for s in live:                                                                     # owners moved along: shared blocks outlive the first of their owners
        L.cml_paged_cache_free_sequence(c, s)
    assert c.contents.free_count == 24


def test_compact_of_nothing_and_refusals(pkg, cache):
    L, c = pkg.lib, cache(4, 2, 4)
    moves = np.zeros(8, np.int32)
    assert L.cml_paged_cache_compact(None, pkg.np_ptr(moves)) == -1 and L.cml_paged_cache_compact(c, None) == -1
    assert L.cml_paged_cache_compact(c, pkg.np_ptr(moves)) == 0
    s = L.cml_paged_cache_init_sequence(c)
    assert L.cml_paged_cache_extend(c, s, 16) == 0 and L.cml_paged_cache_compact(c, pkg.np_ptr(moves)) == 0


def test_caches_with_data(pkg):
    """Forks and compaction of a cache that holds its keys and values on the host move them too."""
    L, rng = pkg.lib, np.random.default_rng(3)
    c = L.cml_paged_kv_cache_create(8, 4, 2, 3)
    size = c.contents.block_size
    rows = rng.standard_normal((3 * size, 2, 2, 3)).astype(np.float32)

    def put(s, r):
        for k, v in r:
            assert L.cml_paged_cache_append(c, s, pkg.np_ptr(np.ascontiguousarray(k)), pkg.np_ptr(np.ascontiguousarray(v))) == 0

    def held(s):
        out = []
        for j in range(c.contents.sequences[s].seq_len):
            b = c.contents.blocks[ids(c, s)[j // size]]
            out.append([[x[(j % size) * 6 + i] for i in range(6)] for x in (b.key_data, b.value_data)])
        return np.array(out, np.float32).reshape(-1, 2, 2, 3)

    gone, s = L.cml_paged_cache_init_sequence(c), None
    put(gone, rows[:size])
    s = L.cml_paged_cache_init_sequence(c)
    put(s, rows[:size + 5])
    child = L.cml_paged_cache_fork(c, s, None, None)
    put(s, rows[size + 5:size + 7])
    put(child, rows[2 * size:2 * size + 3])
    want = {s: rows[:size + 7], child: np.concatenate([rows[:size + 5], rows[2 * size:2 * size + 3]])}
    for _ in range(2):
        for k, w in want.items():
            assert np.array_equal(held(k), w)
        if gone is not None:
            L.cml_paged_cache_free_sequence(c, gone)
            assert L.cml_paged_cache_compact(c, None) == 3 and sorted(set(ids(c, s) + ids(c, child))) == [0, 1, 2]      # (such a cache hands out the highest first)
            gone = None
    L.cml_paged_kv_cache_free(c)


def test_model_calls_without_a_model(pkg):
    L = pkg.lib
    assert L.cml_lm_sequence_fork(None, 0) == -1 and L.cml_lm_compact(None) == -1
    assert L.cml_lm_step_scored(None, None, 0, None, 0, None, None, None, None) == -1


@pytest.mark.parametrize("cache", [-1, 3])
def test_unknown_cache_forms(pkg, tmp_path, cache):
    assert not pkg.lib.cml_lm_load(str(tmp_path).encode(), pkg.LMOptions(pkg.DTYPE_BFLOAT16, 64, 1, 0, cache))
    assert pkg.lib.cml_lm_default_options().cache == pkg.CACHE_DEFAULT
