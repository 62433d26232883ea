"""What a serving loop does around the page operators where the list runs out, pages come back by
hand or a row gets shorter, as the caller's contract has it; run over the reference (CPU) and over
the kernels.  The operators come in as functions of plain lists:

  fork(parents, children, lens, table, shares, free, num_free, page) -> table, shares, left, src, dst
  free(rows, lens, table, shares, free, num_free, page) -> shares, free, left
"""
from __future__ import annotations


class Pages:
    """Rows, their table, and the pages that no row holds."""

    def __init__(self, fork, free, rows, columns, pages, page):
        self.fork_op, self.free_op, self.page = fork, free, page
        self.table, self.lens = [[-1] * columns for _ in range(rows)], [0] * rows
        self.shares, self.free, self.num = [0] * pages, [(7 * i) % pages for i in range(pages)], pages

    def pages_of(self, n):
        return -(-n // self.page)

    def grow(self, row, n):
        """As a step's tables do: a row keeps the pages of its tokens, and takes those that it needs more."""
        for c in range(self.pages_of(self.lens[row]), self.pages_of(n)):
            self.num -= 1
            self.table[row][c] = self.free[self.num]
        self.lens[row] = n

    def fork(self, parents, children, took):
        self.table, self.shares, left, src, dst = self.fork_op(parents, children, self.lens, self.table, self.shares, self.free, self.num, self.page)
        if took(left):
            self.num = left
        return left, src, dst

    def release(self, rows):
        self.shares, self.free, self.num = self.free_op(rows, self.lens, self.table, self.shares, self.free, self.num, self.page)
        for row in rows:
            self.lens[row] = 0

    def add_up(self):
        """Every page is held or on the list, none both or twice, and the counts are the holders'."""
        held = [p for row, n in zip(self.table, self.lens) for p in row[:self.pages_of(n)]]
        free = list(self.free[:max(self.num, 0)])
        assert min(held + free + [0]) >= 0
        assert len(set(free)) == len(free) and not set(held) & set(free), "a page is free twice, or held and free"
        assert set(held) | set(free) == set(range(len(self.shares))), "a page is lost"
        assert list(self.shares) == [max(held.count(p) - 1, 0) for p in range(len(self.shares))]


def refused_fork_and_retry(fork, free, took=lambda left: left >= 0):
    """A fork that finds too few pages is not taken: `num_free` stays the list's count and the
    children's lengths stay as they are; with pages returned the same fork goes through."""
    s = Pages(fork, free, rows=8, columns=5, pages=12, page=16)
    s.grow(0, 40), s.grow(1, 50), s.grow(2, 40)  # 3 + 4 + 3 pages, 2 are left
    s.add_up()
    before = ([list(r) for r in s.table], list(s.shares), s.num)
    left, src, dst = s.fork([0, 1, 0], [4, 5, 6], took)
    assert left == -1 and list(src) == list(dst) == [-1] * 3
    s.add_up()
    assert ([list(r) for r in s.table], list(s.shares), s.num) == before
    s.release([2])
    s.add_up()
    assert s.num == 5
    left, src, dst = s.fork([0, 1, 0], [4, 5, 6], took)
    assert left == 2 and min(dst) >= 0
    for parent, child in zip([0, 1, 0], [4, 5, 6]):
        s.lens[child] = s.lens[parent]
    s.add_up()
    s.release([0, 1, 4, 5, 6])
    s.add_up()
    assert s.num == 12


def pages_back_beside_forked_rows(fork, free, by_hand=lambda s, row: False):
    """Rows that end beside rows forked from them: their shared pages stay off the list.  `by_hand` may
    return a row's pages itself, where it says so."""
    s = Pages(fork, free, rows=6, columns=4, pages=16, page=16)
    s.grow(0, 40), s.grow(1, 32)
    s.fork([0, 1], [2, 3], took=lambda left: True)
    s.lens[2], s.lens[3] = 40, 32
    s.add_up()
    for row in (0, 3, 1):
        if by_hand(s, row):
            s.lens[row] = 0
        else:
            s.release([row])
        s.add_up()
    s.grow(4, 60)  # takes none of row 2's pages
    s.add_up()
    s.release([2, 4])
    s.add_up()
    assert s.num == 16


def rows_that_get_shorter(fork, free, give_back=True):
    """Guessed tokens that are not taken: the pages behind the tokens that a row keeps go back to the
    list, through the operator that frees rows, as the pages of a table of their own."""
    s = Pages(fork, free, rows=6, columns=6, pages=24, page=8)
    for row, n in enumerate((20, 8, 0, 17)):
        s.grow(row, n)
    s.fork([0, 1], [4, 5], took=lambda left: True)
    s.lens[4], s.lens[5] = 20, 8
    s.add_up()
    for grown, kept in (((37, 9, 16, 18, 24, 33), (24, 8, 1, 18, 21, 30)),   # across page borders, within pages, all of them
                        ((40, 8, 1, 25, 25, 31), (24, 8, 0, 17, 21, 30)),
                        ((24, 8, 0, 17, 21, 30), (8, 0, 0, 17, 21, 30))):    # into pages that other rows share
        for row, n in enumerate(grown):
            s.grow(row, n)
        s.add_up()
        first = [s.pages_of(n) for n in kept]
        behind = [[row[min(f + c, len(row) - 1)] for c in range(len(row))] for row, f in zip(s.table, first)]
        more = [(s.pages_of(n) - f) * s.page for n, f in zip(s.lens, first)]
        if give_back:
            s.shares, s.free, s.num = s.free_op(list(range(6)), more, behind, s.shares, s.free, s.num, s.page)
        s.lens = list(kept)
        s.add_up()
    s.release(list(range(6)))
    s.add_up()
    assert s.num == 24
