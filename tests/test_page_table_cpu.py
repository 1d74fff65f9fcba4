"""CPU suite: the bookkeeping of a cache in pages, against a model that keeps every sequence's tokens apart."""
import random

import pytest

from llama3_np_b200 import PageTable


class Model:
    """Page contents as tokens: what the copies and writes of a real cache would leave in the pages."""

    def __init__(self, table):
        self.t, self.size = table, table.page_size
        self.pages = [[None] * self.size for _ in range(table.pages)]
        self.want = {}

    def copy(self, pairs):
        src, dst = [a for a, _ in pairs], [b for _, b in pairs]
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)      # what copy_pages asks for
        for a, b in pairs:
            self.pages[b] = list(self.pages[a])

    def write(self, seq, start, tokens):
        row = self.t.pages_of(seq)
        for i, x in enumerate(tokens):
            self.pages[row[(start + i) // self.size]][(start + i) % self.size] = x
        self.want[seq] = self.want[seq][:start] + tokens

    def check(self):
        used = set()
        for seq, want in self.want.items():
            row = self.t.pages_of(seq)
            assert self.t.length(seq) == len(want) and len(row) == -(-len(want) // self.size)
            assert [self.pages[row[i // self.size]][i % self.size] for i in range(len(want))] == want
            used |= set(row)
        assert self.t.free_pages == self.t.pages - len(used)


@pytest.mark.parametrize("size,pages", [(1, 40), (4, 12), (16, 9), (8, 3)])
def test_random_programs(size, pages):
    rng = random.Random(size * 100 + pages)
    for _ in range(60):
        t = PageTable(pages, size)
        m, names = Model(t), iter(range(10 ** 9))
        for _ in range(40):
            live = list(m.want)
            what = rng.choice(["open", "grow", "grow", "grow", "fork", "fork", "free", "compact"])
            if what == "open" or not live:
                m.want[t.open()] = []
            elif what == "fork":
                s = rng.choice(live)
                m.want[t.fork(s)] = list(m.want[s])
            elif what == "free":
                s = rng.choice(live)
                t.free(s)
                del m.want[s]
                assert s not in t
            elif what == "compact":
                m.copy(t.compact())
                assert all(p < t.pages - t.free_pages for s in m.want for p in t.pages_of(s))
            else:
                some = rng.sample(live, rng.randint(1, len(live)))
                more = [rng.randint(0, 2 * size) for _ in some]
                before = {s: (t.pages_of(s), t.length(s)) for s in live}
                try:
                    m.copy(t.grow(some, more))
                except RuntimeError:
                    assert {s: (t.pages_of(s), t.length(s)) for s in live} == before
                    continue
                for s, n in zip(some, more):
                    m.write(s, len(m.want[s]), [next(names) for _ in range(n)])
            m.check()
        for s in list(m.want):
            t.free(s)
        assert t.free_pages == pages


def test_a_shared_page_is_copied_for_all_but_its_last_sharer():
    t = PageTable(4, 8)
    a = t.open()
    assert t.grow([a], 3) == []
    b, c = t.fork(a), t.fork(a)
    assert t.grow([b, c, a]) == [(0, 1), (0, 2)] and t.free_pages == 1
    assert t.grow([a, b, c], [0, 0, 0]) == []
    t.free(a)
    assert t.compact() == [(2, 0)] and t.pages_of(c) == [0]


def test_refusals():
    for args in [(0, 16), (4, 12), (4, 0), (4, 1 << 17)]:
        with pytest.raises(ValueError):
            PageTable(*args)
    t = PageTable(2, 4)
    a = t.open()
    for call in (lambda: t.grow([a, a]), lambda: t.grow([a], [1, 2]), lambda: t.grow([a], -1), lambda: t.grow([7]), lambda: t.free(7),
                 lambda: t.fork(7), lambda: t.length(7), lambda: t.pages_of(7)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="out of pages"):
        t.grow([a], 9)
    assert t.length(a) == 0 and t.free_pages == 2
