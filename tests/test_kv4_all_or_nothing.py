"""Calls of the 4-bit cache that fail change nothing: no page is lost, no sequence half done."""
import pytest

import b200attn
from b200attn.kv4 import KV4Cache, OutOfPages


def cache(pages=8):
    """A cache on the CPU: accounting works, copies of pages are refused by the library."""
    return KV4Cache(2, 1, pages, device="cpu")


def state(c):
    t = c.tables
    return (sorted(t._free), list(t._uses), {s: list(p) for s, p in t._pages.items()}, dict(t._length))


def test_add_takes_all_or_none():
    c = cache()
    before = state(c)
    for bad in ([64, -1], [-1000, 600], [64, "x"], [64, None]):
        with pytest.raises((ValueError, TypeError)):
            c.add(bad)
        assert state(c) == before, bad
    with pytest.raises(OutOfPages):
        c.add([64 * 8, 1])
    assert state(c) == before
    assert len(c.add([64, 0, 65])) == 3 and c.tables.free_pages == 5


def test_fork_and_free_take_all_or_none():
    c = cache()
    a, b = c.add([100, 64])
    before = state(c)
    with pytest.raises(KeyError):
        c.fork([a, 77])
    assert state(c) == before
    for wrong in ([a, 77], [a, b, 77]):
        with pytest.raises(KeyError):
            c.free(wrong)
        assert state(c) == before
    with pytest.raises(ValueError):
        c.free([a, b, a])
    assert state(c) == before
    x, y = c.fork([a, a])
    c.free([a, x, y, b])
    assert c.tables.free_pages == 8


def test_extend_whose_copies_fail():
    c = cache()
    a, = c.add([100])
    f, g = c.fork([a, a])
    before = state(c)
    with pytest.raises(ValueError, match="CUDA"):
        c.extend([f, a], [30, 200])        # f's last page is shared: a copy
    assert state(c) == before
    with pytest.raises(ValueError, match="CUDA"):
        c.extend([a, f, g], [1, 1, 1])     # two copies, one keeps the page
    assert state(c) == before
    c.free([f, g])
    c.extend([a], [30])                    # nothing to copy
    assert c.tables.length(a) == 130 and c.tables.free_pages == 5


def test_compact_whose_copies_fail():
    c = cache()
    seqs = c.add([64, 64, 64])
    c.free(seqs[:1])
    before = state(c)
    with pytest.raises(ValueError, match="CUDA"):
        c.compact()
    assert state(c) == before
    assert [c.tables.pages(s) for s in seqs[1:]] == [[1], [2]]


def test_copies_are_made_before_the_tables_change(monkeypatch):
    c = cache()
    a, = c.add([100])
    f, = c.fork([a])
    seen = []
    monkeypatch.setattr(b200attn, "kv4_copy_pages",
                        lambda pool, src, dst: seen.append((list(src), list(dst), c.tables.pages(f))))
    c.extend([f], [5])
    assert seen == [([1], [2], [0, 1])] and c.tables.pages(f) == [0, 2] and c.tables.pages(a) == [0, 1]
    c.free([a])
    seen.clear()
    assert c.compact() == 1
    assert seen == [([2], [1], [0, 2])] and c.tables.pages(f) == [0, 1]
