"""PagedCache.table and .tables beside other threads that change the sequences,
against the HIP stand-in of tests/fakehip."""
import threading

import numpy as np
import pytest

from test_attn_host import L  # noqa: F401  (the fixture)


class Between:
    """The library, with something done after the n-th call of seq_tables: what another
    thread may do there."""

    def __init__(self, lib, n, what):
        self.lib, self.left, self.what = lib, n, what

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def sllm_gfx950_seq_tables(self, *args):
        st = self.lib.sllm_gfx950_seq_tables(*args)
        self.left -= 1
        if self.left == 0:
            self.what()
        return st


@pytest.fixture
def cache(amd, L, monkeypatch):  # noqa: F811
    monkeypatch.setattr(amd, "_lib", L)
    c = amd.PagedCache(None, 1, 1, 8, 16, 2000)
    yield c
    c.close()


def grow(c, s, n):
    c.batch([s], [n], 1).close()


@pytest.mark.parametrize("first,then", [(20, 700), (700, 20), (0, 16), (16, 0), (16, 16 * 1000), (16 * 1000, 0)])
def test_a_sequence_that_changes_between_two_calls(amd, L, cache, monkeypatch, first, then):  # noqa: F811
    """The table is the sequence's before the change or after it, whole; never what lay
    in the memory it is returned in."""
    empty = np.empty
    monkeypatch.setattr(amd.np, "empty", lambda n, t: np.full_like(empty(n, t), -77))
    for call in range(1, 4):
        for get in (cache.table, lambda s: cache.tables([s])[0], lambda s: cache.tables([s, s])[1]):
            s = cache.new()
            grow(cache, s, first)
            was = cache.table(s)

            def change(s=s):
                if then > first:
                    grow(cache, s, then - first)
                else:
                    cache.truncate(s, then)

            monkeypatch.setattr(amd, "_lib", Between(L, call, change))
            got = get(s)
            monkeypatch.setattr(amd, "_lib", L)
            now = cache.table(s)
            assert any(np.array_equal(got, x) for x in (was, now)), (call, got[:5], len(got), len(was), len(now))
            cache.free([s])


def test_tables_beside_a_thread(amd, cache):
    """Tables of a sequence whose pages are its numbers in order, while another thread
    makes it longer and shorter."""
    s = cache.new()
    stop = threading.Event()

    def change():
        r = np.random.RandomState(1)
        while not stop.is_set():
            grow(cache, s, int(r.randint(50, 900)))
            cache.truncate(s, int(r.randint(0, 50)))

    t = threading.Thread(target=change)
    t.start()
    try:
        for _ in range(4000):
            got = cache.table(s)
            assert np.array_equal(got, np.arange(len(got)))
    finally:
        stop.set()
        t.join()


def test_tables_of_several(amd, cache):
    a, b, c = cache.new(), cache.new(), cache.new()
    grow(cache, a, 33)
    grow(cache, b, 48)
    assert cache.tables([a, b]).tolist() == [[0, 1, 2], [3, 4, 5]] and cache.table(b).tolist() == [3, 4, 5]
    assert cache.tables([]).shape == (0, 0) and cache.tables([c, c]).shape == (2, 0) and cache.table(c).size == 0
    with pytest.raises(amd.GFX950Error):
        cache.table(77)
    with pytest.raises(ValueError):                     # 3 and 0 pages
        cache.tables([a, c])
    got = cache.table(a)
    got[0] = 9                                          # (the caller's own)
    assert cache.table(a).tolist() == [0, 1, 2] and got.dtype == np.int32


def test_sequence_numbers_of_any_kind(amd, cache):
    """Lists, tuples, ranges and arrays of numpy; none; what is no sequence number."""
    s = [cache.new() for _ in range(4)]
    grow(cache, s[1], 20)
    for kind in (list, tuple, np.array, lambda x: np.array(x, np.int64), iter):
        out = cache.copy(kind(s[:2]))
        assert len(out) == 2 and cache.length(out[1]) == 20
        cache.free(kind(out))
    assert cache.copy([]) == [] and cache.free([]) is None
    with pytest.raises(OverflowError):
        cache.free([1 << 32])                           # (not sequence 0)
    with pytest.raises(TypeError):
        cache.free([1.5])
    with pytest.raises(amd.GFX950Error):
        cache.free([s[0], 9])
    assert cache.length(s[0]) == 0
