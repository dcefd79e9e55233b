"""Sequences of a paged cache that are cut short: the bookkeeping, on the host alone."""
import pytest

from test_paged_fork_cpu import cache, fork, ids  # noqa: F401 (cache is a fixture)


@pytest.mark.parametrize("tokens", [0, 1, 4, 5, 8, 11])
def test_every_length(pkg, cache, tokens):  # noqa: F811
    for length in range(tokens + 1):
        L, c = pkg.lib, cache()
        s = L.cml_paged_cache_init_sequence(c)
        assert L.cml_paged_cache_extend(c, s, tokens) == 0
        had = ids(c, s)
        assert L.cml_paged_cache_truncate(c, s, length) == 0
        keep = -(-length // 4)
        assert ids(c, s) == had[:keep] and c.contents.sequences[s].seq_len == length and c.contents.free_count == 12 - keep
        assert L.cml_paged_cache_extend(c, s, 9) == 0 and ids(c, s)[:keep] == had[:keep] and len(ids(c, s)) == -(-(length + 9) // 4)
        L.cml_paged_cache_free_sequence(c, s)
        assert c.contents.free_count == 12 and sorted(c.contents.free_list[i] for i in range(12)) == list(range(12))


def test_refused(pkg, cache):  # noqa: F811
    L, c = pkg.lib, cache()
    s = L.cml_paged_cache_init_sequence(c)
    assert L.cml_paged_cache_extend(c, s, 10) == 0
    child = fork(pkg, c, s)[0]
    before = (ids(c, s), ids(c, child), c.contents.free_count)
    for who, length in ((s, 11), (s, -1), (s, 7), (s, 1), (child, 5), (child, 3), (9, 0), (-1, 0), (4, 0)):
        assert L.cml_paged_cache_truncate(c, who, length) == -1
    assert L.cml_paged_cache_truncate(None, s, 1) == -1
    assert (ids(c, s), ids(c, child), c.contents.free_count) == before
    # at the border of shared blocks, and inside one's own
    assert L.cml_paged_cache_truncate(c, s, 9) == 0 and L.cml_paged_cache_truncate(c, s, 8) == 0
    assert L.cml_paged_cache_truncate(c, child, 4) == 0 and ids(c, child) == before[1][:1]
    assert L.cml_paged_cache_extend(c, child, 1) == 0 and not set(ids(c, child)[1:]) & set(ids(c, s))
    L.cml_paged_cache_free_sequence(c, s)
    assert L.cml_paged_cache_truncate(c, child, 2) == 0                   # nobody else's by now
    # blocks let go of
    t = L.cml_paged_cache_init_sequence(c)
    assert L.cml_paged_cache_extend(c, t, 20) == 0
    L.cml_paged_cache_release_between(c, t, 0, 13)
    assert ids(c, t)[:3] == [-1, -1, -1]
    free = c.contents.free_count
    assert L.cml_paged_cache_truncate(c, t, 10) == -1 and c.contents.free_count == free
    assert L.cml_paged_cache_truncate(c, t, 13) == 0 and c.contents.free_count == free + 1
    L.cml_paged_cache_free_sequence(c, t)


def test_caches_with_data(pkg):
    c = pkg.lib.cml_paged_kv_cache_create(4, 2, 1, 8)
    s = pkg.lib.cml_paged_cache_init_sequence(c)
    assert pkg.lib.cml_paged_cache_truncate(c, s, 0) == -1
    pkg.lib.cml_paged_kv_cache_free(c)
