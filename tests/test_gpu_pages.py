"""The tables and pages of the paged cache: room, forks, cuts, compaction and copies, against lists."""
import ctypes as C

import numpy as np
import pytest

from serve import PAGE, Lists

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


class Pool:
    """Tables with a small cache whose pages hold marks, and lists beside them."""

    def __init__(self, dev, pages, seqs, width, layers=1, hd=8):
        self.dev, self.c, self.p = dev, dev.kv8(pages, layers, 1, hd), dev.pages(pages, seqs, width)
        self.size = dev.lib.l3m_kv8_page_bytes(layers, 1, hd)
        self.want = Lists(pages, seqs, width)
        self.marks = np.random.default_rng(pages).integers(0, 256, (pages, self.size), dtype=np.uint8)
        assert dev.lib.l3m_dev_upload(self.c.mem, C.c_void_p(self.marks.ctypes.data), self.marks.nbytes) == 0

    def check(self):
        self.want.check(self.dev.pages_state(self.p))
        assert np.array_equal(self.dev.get(self.c.mem, self.marks.shape, np.uint8), self.marks)

    def copied(self, pairs):
        self.marks[[b for _, b in pairs]] = self.marks[[a for a, _ in pairs]]

    def grow(self, ids, counts):
        starts = np.cumsum([0] + list(counts))
        pos = self.dev.pages_grow(self.p, self.c, self.dev.batch(starts, ids))
        got = self.want.grow(list(ids) if ids is not None else list(range(len(counts))), counts)
        if got is not None:
            assert list(pos) == got[0]
            self.copied(got[1])
        self.check()
        return got

    def fork(self, a, b):
        self.dev.pages_fork(self.p, a, b)
        self.want.fork(a, b)
        self.check()

    def cut(self, ids, keep=None):
        self.dev.pages_cut(self.p, ids, keep)
        self.want.cut(ids, keep)
        self.check()

    def compact(self):
        self.dev.pages_compact(self.p, self.c)
        moves = self.want.compact()
        self.copied(moves)
        self.check()
        return moves


def test_steps(dev):
    """Prompts, steps over a page's end, forks that share a page and then write behind it, cuts, a pool that fills."""
    o = Pool(dev, 24, 8, 10, layers=3, hd=40)
    o.check()
    o.grow([0, 3, 5], [1, 128, 300])
    o.grow([5, 0], [84, 127])                        # to a page's end
    o.grow([0, 3, 5], [1, 1, 1])                     # the next pages
    o.grow([3, 4], [0, 0])                           # nothing
    o.fork([5, 5, 3], [1, 2, 7])
    assert [len(c) for c in (o.grow([1, 5, 2], [1, 1, 1])[1],)] == [2]     # all holders: the first keeps the page
    o.fork([0], [4])
    assert len(o.grow([4], [2])[1]) == 1             # one of two: a copy
    assert len(o.grow([0], [2])[1]) == 0             # the other is alone by now
    o.cut([2, 1], [200, 0])
    o.cut([5])
    assert len(o.grow([2, 7], [10, 100])[1]) == 1    # 7's second page is 3's too; 2's is its own
    assert o.compact()
    assert not o.compact()
    o.cut([0, 2, 3, 4, 7])
    assert o.want.refs == [0] * 24


def test_whole_pages_shared(dev):
    """A fork at a page's end shares whole pages only: both go on in new ones and nothing is copied. A copy into another width of layers."""
    o = Pool(dev, 12, 3, 6)
    o.grow([0], [256])
    o.fork([0, 0], [1, 2])
    assert o.grow([2, 0, 1], [1, 1, 129])[1] == []
    o.cut([0, 1, 2], [256, 256, 256])
    o.cut([1], [130])                                # inside a page that all hold
    assert len(o.grow([1], [1])[1]) == 1


def test_failures_change_nothing(dev):
    """Too few pages, too long, bad numbers, the same one twice: nothing changes, the state says why, and until it is cleared nothing is done."""
    o = Pool(dev, 6, 4, 4)
    o.grow([0, 1], [200, 10])
    for state, ids, counts in (("full", [2, 3, 0], [128, 385, 100]), ("long", [0, 1], [313, 1]), ("bad", [4], [1]), ("bad", [-1], [1]), ("bad", [2, 2], [1, 1])):
        o.grow(ids, counts)
        assert o.want.state == state
        o.grow([2], [1])
        o.fork([0], [3])
        o.cut([0])
        o.compact()
        dev.pages_clear(o.p)
        o.want.state = "ok"
        o.check()
    for a, b in (([0], [1]), ([0], [4]), ([9], [2]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([2], [2]), ([-1], [2])):
        o.fork(a, b)
        assert o.want.state == "bad"
        dev.pages_clear(o.p)
        o.want.state = "ok"
    for ids, keep in (([0], [201]), ([0], [-1]), ([4], None), ([0, 0], None), ([2], [1])):
        o.cut(ids, keep)
        assert o.want.state == "bad"
        dev.pages_clear(o.p)
        o.want.state = "ok"
    o.grow([2, 3], [128, 256])                       # just fits
    o.grow([1], [119])
    assert o.want.state == "full"
    assert dev.lib.l3m_k_pages_reset(C.byref(o.p), None) == 0
    o.want = Lists(6, 4, 4)
    o.check()


def test_odd_batches(dev):
    """ids None; starts that go down or past the rows are brought into order; an empty list."""
    o = Pool(dev, 10, 4, 4)
    o.grow(None, [3, 0, 200])
    dev.pages_grow(o.p, o.c, dev.batch([0, 5, 2, 99, 7], [0, 1, 2, 3], n=8))       # rows 0 .. 4, none, 5 .. 7 from the third's start, none
    assert list(dev.pages_state(o.p)["len"]) == [8, 0, 206, 0]
    assert dev.lib.l3m_k_pages_grow(C.byref(o.p), C.byref(o.c), C.byref(dev.batch([0])), None, None) == 0
    assert dev.lib.l3m_k_pages_fork(C.byref(o.p), None, None, 0, None) == 0 and dev.lib.l3m_k_pages_cut(C.byref(o.p), None, None, 0, None) == 0
    assert dev.pages_state(o.p)["state"] == "ok"


@pytest.mark.parametrize("pages, seqs, width, seed", [(3000, 1500, 4, 0), (5000, 40, 200, 1), (1025, 1024, 3, 2), (300, 100, 40, 3), (64, 16, 8, 4)])
def test_many(dev, pages, seqs, width, seed):
    """Random calls over many sequences and pages, more than the planning workgroup's threads."""
    o, rng = Pool(dev, pages, seqs, width), np.random.default_rng(seed)
    for _ in range(12):
        what = rng.choice(["grow", "grow", "fork", "cut", "compact"])
        n = int(rng.integers(1, seqs + 1))
        ids = [int(i) for i in rng.permutation(seqs)[:n]]
        if what == "grow":
            room = [width * PAGE - o.want.len[i] for i in ids]
            counts = [int(min(r, rng.choice([0, 1, 1, rng.integers(0, 2 * PAGE)]))) for r in room]
            if n <= 8:
                counts[0] = room[0]
            o.grow(ids, counts)
        elif what == "fork":
            empty = [i for i in range(seqs) if not o.want.len[i]]
            full = [i for i in range(seqs) if o.want.len[i]]
            if empty and full:
                to = empty[:int(rng.integers(1, len(empty) + 1))]
                o.fork([int(rng.choice(full)) for _ in to], to)
        elif what == "cut":
            o.cut(ids, [int(rng.integers(0, o.want.len[i] + 1)) for i in ids] if rng.random() < 0.7 else None)
        else:
            o.compact()
        if o.want.state != "ok":
            dev.pages_clear(o.p)
            o.want.state = "ok"


def test_rows_outside_lists(dev):
    """A cache of more pages than the tables count: the rest is never touched."""
    dev_c, p = dev.kv8(9, 1, 1, 8), dev.pages(4, 2, 4)
    size = dev.lib.l3m_kv8_page_bytes(1, 1, 8)
    marks = np.random.default_rng(1).integers(0, 256, (9, size), dtype=np.uint8)
    assert dev.lib.l3m_dev_upload(dev_c.mem, C.c_void_p(marks.ctypes.data), marks.nbytes) == 0
    dev.pages_grow(p, dev_c, dev.batch([0, 200], [0]))
    dev.pages_fork(p, [0], [1])
    dev.pages_grow(p, dev_c, dev.batch([0, 1], [1]))
    got = dev.get(dev_c.mem, marks.shape, np.uint8)
    assert np.array_equal(got[2], marks[1]) and np.array_equal(got[3:], marks[3:]) and list(dev.pages_state(p)["refs"]) == [2, 1, 1, 0]
