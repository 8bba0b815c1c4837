"""Whether a step of forked requests fits the pool: what `Engine.check_step` says against the step's own bookkeeping (no GPU)."""
import types

import numpy as np
import pytest

from hk_b200.cache import CacheBooks, OutOfPages
from hk_b200.engine import Engine, StepEntry


def engine(books):
    """An engine without a model: what `check_step` looks at."""
    eng = Engine.__new__(Engine)
    eng.cache = types.SimpleNamespace(books=books)
    eng.vocab, eng.max_batch_tokens, eng.takes_trees = 100, 1000, True
    eng._requests, eng._trees = {s: s for s in range(books.max_requests)}, {}
    return eng


def run(books, lens):
    """A step's bookkeeping, in the engine's order: {slot: new tokens}."""
    for s in lens:
        books.release_passed(s)
    for s, n in lens.items():
        books.extend(s, n)


def test_a_page_that_two_windows_pass_in_one_step():
    books = CacheBooks([4], page_tokens=4, num_pages=3, max_requests=2, max_context=64)
    a = books.open()
    books.extend(a, 8)
    b = books.fork(a)                          # pages 0 and 1 held by both, 0 passed by both windows; one is free, two are needed
    engine(books).check_step([StepEntry(a, [1], []), StepEntry(b, [1], [])])
    run(books, {a: 1, b: 1})
    books.audit()
    assert books.free_pages() == [0]


def test_a_page_that_one_request_passes_and_another_writes():
    books = CacheBooks([4], page_tokens=4, num_pages=4, max_requests=3, max_context=64)
    a = books.open()
    books.extend(a, 2)
    b = books.fork(a)
    books.extend(b, 6)                         # b's first page is its own copy
    books.close(b)
    b = books.fork(a)
    books.release_passed(b)
    books.truncate(a, 1)
    c = books.open()
    books.extend(c, 12)                        # the pool's last pages
    assert books.free_pages() == [0]
    with pytest.raises(OutOfPages):            # both write the shared page: one copy is needed
        engine(books).check_step([StepEntry(a, [1], []), StepEntry(b, [1], [])])
    # c's window gives its first pages back in the same step
    engine(books).check_step([StepEntry(a, [1], []), StepEntry(b, [1], []), StepEntry(c, [1], [])])
    run(books, {a: 1, b: 1, c: 1})
    books.audit()


@pytest.mark.parametrize("seed", range(12))
def test_what_is_refused_would_not_have_fitted(seed):
    """Random forks and steps in a small pool: `check_step` raises exactly where the bookkeeping would."""
    rng = np.random.default_rng(seed)
    page = int(rng.choice([1, 2, 4]))
    windows = [[None], [int(rng.integers(2, 9))], [None, int(rng.integers(2, 9))]][seed % 3]
    books = CacheBooks(windows, page_tokens=page, num_pages=int(rng.integers(5, 11)), max_requests=5, max_context=60)
    eng, live, refused, tight = engine(books), [], 0, 0
    for _ in range(500):
        op = rng.random()
        if op < 0.1 and len(live) < 5:
            live.append(books.open())
        elif op < 0.3 and live and len(live) < 5:
            live.append(books.fork(int(rng.choice(live))))
        elif op < 0.4 and live:
            books.close(live.pop(int(rng.integers(0, len(live)))))
        elif live:
            some = [int(s) for s in rng.permutation(live)[:int(rng.integers(1, len(live) + 1))]]
            lens = {s: (int(rng.integers(1, 6)) if rng.random() < 0.3 else 1) for s in some}
            lens = {s: n for s, n in lens.items() if int(books.length[s]) + n <= 60}
            if not lens:
                continue
            before = books.free_pages()
            try:
                eng.check_step([StepEntry(s, [1] * n, []) for s, n in lens.items()])
            except OutOfPages:
                refused += 1
                with pytest.raises(OutOfPages):        # from here on the books are half through a step: begin anew
                    run(books, lens)
                for s in live:
                    books.close(s)
                books.take_copies()
                live = []
                books.audit()
                continue
            run(books, lens)
            books.take_copies()
            books.audit()
            tight += min(books.free_pages()) == 0 < min(before)
    assert refused > 0 and tight > 0


def test_steps_without_forks_ask_for_no_copies(monkeypatch):
    import torch

    from hk_b200.cache.device import PagedCache
    from hk_b200.parts.base import KVCacheSpec, Precision
    cache = PagedCache([KVCacheSpec(2, 4)], Precision(torch.float32, torch.device("cpu")), 4, 8, 3, 32)
    taken = []
    take = cache.books.take_copies
    monkeypatch.setattr(cache.books, "take_copies", lambda: taken.append(1) or take())
    a = cache.open()
    for n in (6, 1, 1):
        cache.books.extend(a, n)
        cache.sync_tables()
    assert not taken
    cache.books.extend(cache.fork([a])[0], 1)          # at a full page: no copy either
    cache.sync_tables()
    assert not taken
    cache.books.extend(a, 1)
    cache.books.extend(cache.fork([a])[0], 1)
    cache.sync_tables()
    assert taken == [1] and not cache.books.owes_copies()
