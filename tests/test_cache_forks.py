"""Forked requests in the cache's books: shared pages, copies before a write, nothing lost or given back while it is read (no GPU)."""
import numpy as np
import pytest
import torch

from hk_b200.cache import CacheBooks, CacheError, OutOfPages, TooManyRequests


def test_a_fork_shares_pages_until_one_of_the_two_writes():
    books = CacheBooks([None], page_tokens=4, num_pages=8, max_requests=3, max_context=32)
    a = books.open()
    books.extend(a, 6)                       # page 0 full, page 1 half
    b = books.fork(a)
    t = books.groups[0].table
    assert (t[a, :2] == t[b, :2]).all() and books.free_pages() == [6] and int(books.length[b]) == 6
    books.audit()
    assert books.pages_to_take(b, 1) == [1] and books.shared_pages(b) == [(int(t[a, 1]), 2)]
    books.extend(b, 1)                       # b writes row 2 of page 1: a page of its own
    assert t[b, 0] == t[a, 0] and t[b, 1] != t[a, 1]
    assert books.take_copies().tolist() == [[0, int(t[a, 1]), int(t[b, 1]), 2]] and len(books.take_copies()) == 0
    assert books.shared_pages(a) == [(-1, 0)] and books.pages_to_take(a, 1) == [0]
    books.extend(a, 1)                       # a holds its page alone now
    assert len(books.take_copies()) == 0
    books.audit()
    books.close(a)
    assert books.free_pages() == [8 - 2]     # b's two; page 0 went on with b
    books.audit()
    books.close(b)
    assert books.free_pages() == [8]
    with pytest.raises(CacheError):
        books.fork(a)


def test_a_fork_at_a_full_page_copies_nothing():
    books = CacheBooks([None, None], page_tokens=4, num_pages=6, max_requests=4, max_context=32)
    a = books.open()
    books.extend(a, 8)
    b, c = books.fork(a), books.fork(a)
    for s in (a, b, c):
        books.extend(s, 1)
    assert len(books.take_copies()) == 0 and books.free_pages() == [1, 1]
    books.audit()


def test_errors_leave_everything_as_it_was():
    books = CacheBooks([None], page_tokens=4, num_pages=2, max_requests=2, max_context=32)
    a = books.open()
    books.extend(a, 6)
    b = books.fork(a)
    with pytest.raises(TooManyRequests):
        books.fork(a)
    before = books.groups[0].table.copy()
    with pytest.raises(OutOfPages):
        books.extend(b, 1)                   # no page for the copy
    assert (books.groups[0].table == before).all() and int(books.length[b]) == 6 and len(books.take_copies()) == 0
    books.audit()
    books.close(a)
    books.extend(b, 1)                       # alone now: in place
    assert len(books.take_copies()) == 0
    books.audit()


def test_a_window_passes_a_shared_page_for_each_holder():
    books = CacheBooks([6], page_tokens=4, num_pages=8, max_requests=2, max_context=64)
    a = books.open()
    books.extend(a, 10)
    b = books.fork(a)
    for _ in range(3):
        books.extend(a, 4)
        books.audit()
    # a has passed pages that b still reads: they are not in the pool
    free = books.free_pages()[0]
    held = [int(p) for p in books.groups[0].table[b] if p >= 0]
    assert books.pages_passed(a)[0] <= 1 and free == 8 - len(set(held) | {int(p) for p in books.groups[0].table[a] if p >= 0})
    books.close(b)
    books.audit()


def test_truncated_into_a_shared_page():
    books = CacheBooks([None], page_tokens=4, num_pages=8, max_requests=2, max_context=64)
    a = books.open()
    books.extend(a, 12)
    b = books.fork(a)
    books.truncate(b, 5)                     # inside page 1, which a reads on to its end
    books.audit()
    books.extend(b, 1)
    copies = books.take_copies().tolist()
    assert copies == [[0, int(books.groups[0].table[a, 1]), int(books.groups[0].table[b, 1]), 1]]
    books.audit()


@pytest.mark.parametrize("seed", range(8))
def test_random_forks_against_plain_contents(seed):
    """What every request reads, followed in a plain model of the pages: a write never shows in another request."""
    rng = np.random.default_rng(seed)
    page = int(rng.choice([1, 3, 4, 8]))
    windows = [None, int(rng.integers(2, 20))] if seed % 2 else [None]
    books = CacheBooks(windows, page_tokens=page, num_pages=int(rng.integers(12, 60)), max_requests=6, max_context=120)
    pages = [np.full((books.groups[g].pool.num_pages, page), -1, dtype=np.int64) for g in range(len(windows))]
    contents = {}
    stamp = 0
    for _ in range(700):
        op = rng.random()
        try:
            if op < 0.1:
                contents[books.open()] = []
            elif op < 0.25 and contents:
                s = int(rng.choice(list(contents)))
                contents[books.fork(s)] = list(contents[s])
            elif op < 0.35 and contents:
                s = int(rng.choice(list(contents)))
                books.close(s)
                del contents[s]
            elif op < 0.4 and contents and windows == [None]:
                s = int(rng.choice(list(contents)))
                keep = int(rng.integers(0, len(contents[s]) + 1))
                books.truncate(s, keep)
                contents[s] = contents[s][:keep]
            elif contents:
                s = int(rng.choice(list(contents)))
                n = int(rng.integers(1, 12)) if rng.random() < 0.3 else 1
                start = len(contents[s])
                need, free = books.pages_to_take(s, n), books.free_pages()
                passed = books.pages_passed(s)
                books.extend(s, n)
                assert all(k <= f + back for k, f, back in zip(need, free, passed))
                for g, a, b, rows in books.take_copies().tolist():
                    pages[g][b, :rows] = pages[g][a, :rows]
                for i in range(start, start + n):
                    stamp += 1
                    contents[s].append(stamp)
                    for g in range(len(windows)):
                        pages[g][books.groups[g].table[s, i // page], i % page] = stamp
        except (OutOfPages, TooManyRequests):
            pass
        except Exception as e:
            if type(e).__name__ != "ContextFull":
                raise
        books.audit()
        for s, want in contents.items():
            for g, w in enumerate(windows):
                lo = 0 if w is None else max(0, len(want) - w + 1)
                got = [int(pages[g][books.groups[g].table[s, i // page], i % page]) for i in range(lo, len(want))]
                assert got == want[lo:], "a request reads what another wrote"
    for s in list(contents):
        books.close(s)
    books.audit()
    assert all(f == g.pool.num_pages for f, g in zip(books.free_pages(), books.groups))


def test_the_cache_copies_in_order_and_forks_states():
    """Shared pages and states on the CPU's tensors: the copies that the books owe are made in their order."""
    from hk_b200.cache.device import PagedCache
    from hk_b200.parts.base import KVCacheSpec, Precision, StateSpec
    cache = PagedCache([KVCacheSpec(2, 4), StateSpec((3,), torch.float32)], Precision(torch.float32, torch.device("cpu")), 4, 6, 3, 32)
    a = cache.open()
    cache.books.extend(a, 6)
    cache.sync_tables()
    k = cache.layers[0][0].k_pages
    pa = [int(p) for p in cache.books.groups[0].table[a, :2]]
    k[pa[0]], k[pa[1]] = 1.0, 2.0
    cache.layers[1][0].state[a] = 7.0
    b, c = cache.fork([a, a])
    assert (cache.layers[1][0].state[b] == 7.0).all() and (cache.layers[1][0].state[c] == 7.0).all()
    cache.books.extend(b, 1)
    cache.books.extend(c, 1)
    cache.sync_tables()
    for s in (b, c):
        p = int(cache.books.groups[0].table[s, 1])
        assert p != pa[1] and (k[p, :, :2] == 2.0).all()
        assert (cache.tables[0][s, :2] == torch.tensor([pa[0], p], dtype=torch.int32)).all()
    # a copy from a page that an earlier copy of the same call wrote
    first = int(cache.books.groups[0].table[b, 1])
    k[first, :, 2] = 3.0
    cache.books.close(c)
    d = cache.fork([b])[0]
    cache.books.extend(d, 1)
    cache.sync_tables()
    assert (k[int(cache.books.groups[0].table[d, 1]), :, :3] == k[first, :, :3]).all()
    cache.books.audit()
