"""GPU: an assignment for which pages run short, and how a caller goes on."""
from __future__ import annotations

import numpy as np
import pytest

from paged_reference import D

pytestmark = pytest.mark.gpu


class Books:
    def __init__(self, cv, ctx, torch, table, pages, size=16):
        self.ints = lambda v: torch.tensor(np.asarray(v, np.int32), device="cuda")
        self.pool = cv.alloc_pages(cv.PAGE_I8, pages, size, 1)
        self.table, S = self.ints(table), len(table)
        self.keep, self.need, self.refs = self.ints([0] * S), self.ints([0] * S), self.ints([0] * pages)
        self.plan = cv.PageAssigner(ctx, [self.pool], self.table, self.keep, self.need, refs=self.refs)

    def __call__(self, keep, need):
        self.keep.copy_(self.ints(keep)), self.need.copy_(self.ints(need))
        self.plan()
        return self.plan.room.tolist()


def test_those_who_wait_let_the_others_go_on(ctx, cv, cuda):
    """The second asks for more than there is: all behind it are without room, the last too, whose page has some.  Once the second
    waits, the others have theirs."""
    books = Books(cv, ctx, cuda, [[0, -1, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1]], 6)
    keep = [16, 16, 16, 9]
    assert books(keep, [17, 48, 17, 10]) == [17, 16, 16, 9]
    assert books.table.tolist() == [[0, 4, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1]]
    # (16 positions are kept, so the first asks for its second page again)
    assert books(keep, [17, 16, 17, 10]) == [17, 16, 17, 10]
    assert books.table.tolist() == [[0, 4, -1], [1, -1, -1], [2, 5, -1], [3, -1, -1]]
    assert books.refs.tolist() == [1] * 6


def shared(cv, ctx, torch, pages):
    """Three sequences of 9 positions on page 0, and a function that appends a row to some of them."""
    books = Books(cv, ctx, torch, [[0, -1, -1]] * 3, pages)
    rows = torch.randn(1, 9, D, device="cuda")
    cv.PageAppender(ctx, books.pool, rows, rows, books.table[:1], books.ints([0]))()
    new, at, count = torch.randn(3, 1, D, device="cuda"), books.ints([9] * 3), books.ints([0] * 3)
    plan = cv.PageAppender(ctx, books.pool, new, new, books.table, at, n_new=count, refs=books.refs)

    def append(n):
        count.copy_(books.ints(n))
        plan()
        return ctx.sync_status()

    return books, append


def test_one_that_waits_lets_go_of_a_shared_tail(ctx, cv, cuda):
    """The second asks for three of two pages.  The first has room, but may not write while the others hold its page; once the second
    waits, the first and the third get copies."""
    books, append = shared(cv, ctx, cuda, 3)
    assert books([9] * 3, [10, 40, 10]) == [10, 9, 9] and books.refs.tolist() == [3, 0, 0]
    assert append([1, 0, 0]) == (6, 5)
    before = books.pool.k.clone()
    assert books([9] * 3, [10, 9, 10]) == [10, 9, 10] and books.refs.tolist() == [1] * 3
    assert books.table[:, 0].tolist() == [1, 0, 2]
    assert bool((books.pool.k == before[0]).all())
    assert append([1, 0, 1])[0] == 0
    assert bool((books.pool.k[0] == before[0]).all()) and not bool((books.pool.k[1] == before[0]).all())


def test_one_that_ends_lets_go_of_a_shared_tail(ctx, cv, cuda):
    """One page for two copies: the third stays on the first's page.  Where it waits the first would need a page too; where it ends the
    first writes in place."""
    books, append = shared(cv, ctx, cuda, 2)
    assert books([9] * 3, [10] * 3) == [10, 10, 9] and books.refs.tolist() == [2, 1]
    assert append([1, 0, 0]) == (6, 5)
    assert books([9] * 3, [10, 10, 9]) == [9, 9, 9] and books.refs.tolist() == [2, 1]
    assert books([9, 9, 0], [10, 10, 0]) == [10, 10, 0] and books.refs.tolist() == [1, 1]
    assert append([1, 1, 0])[0] == 0
