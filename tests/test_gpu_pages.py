"""Hand-out of a paged cache's pages on a B200 against its definition (oracle/batch.py)."""
import ctypes as C

import numpy as np
import pytest

from oracle import batch as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(gpu_lib):
    from nebula_b200 import lib
    return lib


class Pool:
    def __init__(self, L, rng, seqs, pages, page, table_pages, held):
        order = rng.permutation(pages).astype(np.int32)
        self.L, self.seqs, self.pages, self.page = L, seqs, pages, page
        table = np.full((seqs, table_pages), -7, np.int32)
        at = 0
        for s, h in enumerate(held):
            table[s, :h] = order[at:at + h]
            at += h
        free = np.full(pages, -5, np.int32)
        free[:pages - at] = order[at:]
        self.host = B.Pages(table, held, free[:pages - at], page)
        self.table, self.held, self.free = L.Device(table), L.Device(np.array(held, np.int32)), L.Device(free)
        self.count = L.Device(np.array([pages - at], np.int32))
        self.c = L.PagePool(self.table.p, self.held.p, self.free.p, self.count.p, pages, page, table_pages)

    def same(self):
        np.testing.assert_array_equal(self.held.get(), self.host.held)
        np.testing.assert_array_equal(self.table.get(), self.host.table)
        n = int(self.count.get()[0])
        assert n == len(self.host.stack)
        np.testing.assert_array_equal(self.free.get()[:n], self.host.stack)

    def reserve(self, lengths, counts, tokens, slots=True):
        L, n = self.L, self.seqs
        d, c = L.Device(np.array(lengths, np.int32)), None if counts is None else L.Device(np.array(counts, np.int32))
        s, t = L.Device(np.full((n, tokens), -3, np.int32)), L.Device(np.full(n, -3, np.int32))
        L.call("pages_reserve", C.byref(self.c), s.p if slots else None, t.p, d.p, c.p if c else None, n, tokens)
        taken, want = self.host.reserve(lengths, [tokens] * n if counts is None else counts, tokens, self.pages)
        np.testing.assert_array_equal(t.get(), taken)
        np.testing.assert_array_equal(s.get(), want if slots else np.full((n, tokens), -3))
        self.same()
        return taken

    def release(self, lengths, shared=0):
        L = self.L
        d, f = L.Device(np.array(lengths, np.int32)), L.Device(np.full(self.seqs, -3, np.int32))
        L.call("pages_release", C.byref(self.c), f.p, d.p, shared, self.seqs)
        freed = self.host.release(lengths, shared, self.pages)
        np.testing.assert_array_equal(f.get(), freed)
        self.same()
        return freed


@pytest.mark.parametrize("seqs,tokens,page,longest", [(1, 1, 16, 0), (1, 64, 16, 40), (3, 17, 64, 300), (33, 5, 32, 900), (1024, 1, 16, 200),
                                                      (1000, 64, 256, 3000), (5, 4096, 16, 100), (1, 100000, 16, 7), (257, 17, 128, 500)])
@pytest.mark.parametrize("scarce", [False, True])
def test_steps(L, seqs, tokens, page, longest, scarce):
    """Sequences grow by what a step commits, some end and begin anew, the refused ones wait."""
    rng = np.random.default_rng(seqs + tokens)
    lengths = rng.integers(0, longest + 1, seqs)
    held = -(-lengths // page)
    most = -(-(longest + 4 * tokens) // page)
    wanted = int((-(-(lengths + tokens) // page)).sum())
    pages = max(int(held.sum()), (wanted + int(held.sum())) // 2) if scarce else seqs * most
    p = Pool(L, rng, seqs, max(pages, 1), page, most, held)
    for step in range(4):
        counts = None if step == 1 else [int(c) for c in rng.integers(0, tokens + 1, seqs)]
        full = [tokens] * seqs if counts is None else counts
        taken = p.reserve([int(n) for n in lengths], counts, tokens, slots=step != 2)
        for s in range(seqs):
            if taken[s] >= 0:
                lengths[s] += int(rng.integers(0, full[s] + 1))
        ended = rng.random(seqs) < 0.2
        freed = p.release([-1 if e else int(n) for e, n in zip(ended, lengths)])
        assert min(freed) >= 0
        lengths[ended] = 0
    for s in range(seqs):  # no page is in two places
        lengths[s] = -1
    p.release([int(n) for n in lengths])
    assert sorted(p.host.stack) == list(range(max(pages, 1)))


def test_shared_pages_stay(L):
    rng = np.random.default_rng(1)
    p = Pool(L, rng, 3, 40, 16, 12, [4, 4, 4])
    assert p.release([-1, 20, 64], shared=3) == [1, 1, 0]
    assert p.reserve([48, 50, 64], [3, 0, 1], 3) == [1, 1, 1]


def test_bad_sequences_are_refused_alone(L):
    rng = np.random.default_rng(2)
    p = Pool(L, rng, 6, 60, 16, 5, [1, 1, 1, 1, 1, 1])
    assert p.reserve([16, -1, 80, 16, 0, 79], [2, 2, 1, 4, -1, 1], 3) == [1, -1, -1, -1, -1, 4]
    p.host.held[1] = 6
    p.host.held[3] = -1
    p.held.set(np.array(p.host.held, np.int32))
    assert p.reserve([16, 16, 16, 16, 16, 16], None, 3) == [0, -1, 1, -1, 1, 0]
    assert p.release([0] * 6) == [2, -1, 2, -1, 2, 5]
    p.host.table[0][0] = 60  # outside the pool: no slot
    p.host.table[2][0] = -1
    p.host.held = [1, 0, 1, 0, 0, 0]
    p.table.set(np.array(p.host.table, np.int32))
    p.held.set(np.array(p.host.held, np.int32))
    p.reserve([0, 0, 0, 0, 0, 0], None, 3)


def test_stack_that_cannot_be(L):
    """A height outside the pool counts as empty; pages that would not fit are not taken back."""
    rng = np.random.default_rng(3)
    p = Pool(L, rng, 2, 10, 16, 8, [3, 2])
    for height in (-1, 11, 2 ** 31 - 1):
        p.count.set(np.array([height], np.int32))
        before = p.table.get(), p.held.get(), p.free.get()
        t, n, s = L.Device(np.zeros(2, np.int32)), L.Device(np.array([60, 30], np.int32)), L.Device(np.zeros((2, 4), np.int32))
        L.call("pages_reserve", C.byref(p.c), s.p, t.p, n.p, None, 2, 4)
        assert list(t.get()) == [-2, -2] and (s.get() == -1).all()
        L.call("pages_release", C.byref(p.c), t.p, L.Device(np.array([48, 0], np.int32)).p, 0, 2)
        assert list(t.get()) == [0, -1]
        for a, b in zip(before, (p.table.get(), p.held.get(), p.free.get())):
            np.testing.assert_array_equal(a, b)
        assert p.count.get()[0] == height


def test_captured_steps(L):
    """Reserving, committing and giving back without the host: a graph of both calls, the lengths changed in between."""
    rng = np.random.default_rng(4)
    p = Pool(L, rng, 9, 300, 16, 30, [0] * 9)
    n, c = L.Device(np.zeros(9, np.int32)), L.Device(np.zeros(9, np.int32))
    s, t, f = L.Device(np.zeros((9, 21), np.int32)), L.Device(np.zeros(9, np.int32)), L.Device(np.zeros(9, np.int32))
    g = C.c_void_p()
    L.call("graph_begin", C.byref(g))
    L.call("pages_release", C.byref(p.c), f.p, n.p, 0, 9)
    L.call("pages_reserve", C.byref(p.c), s.p, t.p, n.p, c.p, 9, 21)
    L.call("graph_end", g)
    lengths = [0] * 9
    for _ in range(6):
        counts = [int(x) for x in rng.integers(0, 22, 9)]
        n.set(np.array(lengths, np.int32))
        c.set(np.array(counts, np.int32))
        L.call("graph_launch", g)
        freed = p.host.release(lengths, 0, 300)
        taken, slots = p.host.reserve(lengths, counts, 21, 300)
        np.testing.assert_array_equal(f.get(), freed)
        np.testing.assert_array_equal(t.get(), taken)
        np.testing.assert_array_equal(s.get(), slots)
        p.same()
        lengths = [x + int(rng.integers(0, y + 1)) for x, y in zip(lengths, counts)]
    L.graph_destroy(g)
