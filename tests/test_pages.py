"""The paged cache's host bookkeeping (kernrt_b200/csrc/pages.cpp) without a GPU:
random runs of every operation against a plain model that keeps each
sequence's contents, and the refusals, which change nothing."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
S, U64 = C.c_size_t, C.c_uint64


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("pages") / "pages.so")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", so,
                    os.path.join(ROOT, "tests", "cpp", "pages_driver.cpp"),
                    os.path.join(ROOT, "kernrt_b200", "csrc", "pages.cpp")], check=True)
    lib = C.CDLL(so)
    lib.pm_new.restype = C.c_void_p
    lib.pm_new.argtypes = [S] * 4
    lib.pm_msg.restype = C.c_char_p
    lib.pm_available.restype = S
    lib.pm_compact.restype = S
    for name, args in (("pm_delete", []), ("pm_available", []), ("pm_open", [C.POINTER(U64)]),
                       ("pm_fork", [U64, S, S, C.c_void_p]), ("pm_copy", [U64, S, C.POINTER(U64), C.c_void_p, C.POINTER(S)]),
                       ("pm_trim", [U64, S]), ("pm_close", [C.c_void_p, S]),
                       ("pm_extend", [C.c_void_p, C.c_void_p, S, C.c_void_p, C.POINTER(S)]),
                       ("pm_compact", [C.c_void_p]),
                       ("pm_table", [U64, C.POINTER(S), C.c_void_p, C.POINTER(S), C.POINTER(S)])):
        getattr(lib, name).argtypes = [C.c_void_p] + args
    return lib


class Refused(Exception):
    pass


class Map:
    """The C++ map, with a pool whose contents follow the copies it orders."""

    def __init__(self, lib, pages, page, seqs, length):
        self.lib, self.page, self.n = lib, page, pages
        self.m = lib.pm_new(pages, page, seqs, length)
        self.pool = np.full((pages, page), -1, np.int64)
        self.copies = np.empty((pages + seqs + 1, 3), np.int32)
        self.tables = {}  # as a device would hold them, from the dirty ranges

    def _ok(self, rc):
        if rc:
            raise Refused(rc, self.lib.pm_msg().decode())

    def _copied(self, n):
        for src, dst, rows in self.copies[:n].tolist():
            assert 0 < rows <= self.page
            self.pool[dst, :rows] = self.pool[src, :rows]

    def available(self):
        return self.lib.pm_available(self.m)

    def open(self):
        h = U64()
        self._ok(self.lib.pm_open(self.m, C.byref(h)))
        self.tables[h.value] = []
        return h.value

    def fork(self, seq, length, n):
        out = np.zeros(max(n, 1), np.uint64)
        self._ok(self.lib.pm_fork(self.m, seq, length, n, out.ctypes.data))
        for h in out[:n].tolist():
            self.tables[h] = []
        return out[:n].tolist()

    def copy(self, seq, length):
        h, n = U64(), S()
        self._ok(self.lib.pm_copy(self.m, seq, length, C.byref(h), self.copies.ctypes.data, C.byref(n)))
        self._copied(n.value)
        self.tables[h.value] = []
        return h.value

    def trim(self, seq, length):
        self._ok(self.lib.pm_trim(self.m, seq, length))

    def close(self, seqs):
        a = np.array(seqs, np.uint64)
        self._ok(self.lib.pm_close(self.m, a.ctypes.data, a.size))

    def extend(self, seqs, rows):
        a, r, n = np.array(seqs, np.uint64), np.array(rows, np.uint64), S()
        self._ok(self.lib.pm_extend(self.m, a.ctypes.data, r.ctypes.data, a.size, self.copies.ctypes.data, C.byref(n)))
        self._copied(n.value)

    def compact(self):
        n = self.lib.pm_compact(self.m, self.copies.ctypes.data)
        dst = {d for _, d, _ in self.copies[:n].tolist()}
        assert not dst & {s for s, _, _ in self.copies[:n].tolist()}, "a move reads what another writes"
        self._copied(n)
        return n

    def table(self, seq):
        length, n, dirty = S(), S(), S()
        pages = np.empty(self.n, np.int32)
        self._ok(self.lib.pm_table(self.m, seq, C.byref(length), pages.ctypes.data, C.byref(n), C.byref(dirty)))
        t = self.tables[seq]
        t[dirty.value:] = pages[dirty.value:n.value].tolist()
        assert t[:n.value] == pages[:n.value].tolist(), "an entry changed outside the dirty range"
        del t[n.value:]
        return length.value, t


@pytest.mark.parametrize("seed", range(6))
def test_random_operations_keep_every_sequence(lib, seed):
    rng = random.Random(seed)
    page = rng.choice([1, 2, 4, 16])
    m = Map(lib, 40, page, 9, 40 * page)
    want = {}
    fresh = 0
    refused = 0
    for _ in range(1500):
        op = rng.choice(["open", "extend", "extend", "extend", "extend", "fork", "copy", "trim", "close", "compact"])
        live = list(want)
        try:
            if op == "open":
                want[m.open()] = []
            elif op == "compact":
                used = 40 - m.available()
                m.compact()
                held = {p for q in want for p in m.table(q)[1]}
                assert held == set(range(used))
            elif not live:
                continue
            elif op == "extend":
                some = rng.sample(live, rng.randint(1, len(live)))
                rows = [rng.choice([0, 1, 1, 1, 3, page, 5 * page]) for _ in some]
                m.extend(some, rows)
                for q, n in zip(some, rows):
                    length, t = m.table(q)
                    for i in range(len(want[q]), length):
                        fresh += 1
                        m.pool[t[i // page], i % page] = fresh
                        want[q].append(fresh)
            elif op == "fork":
                q = rng.choice(live)
                n = rng.randint(0, len(want[q]))
                for c in m.fork(q, n, rng.randint(0, 3)):
                    want[c] = want[q][:n]
            elif op == "copy":
                q = rng.choice(live)
                n = rng.randint(0, len(want[q]))
                want[m.copy(q, n)] = want[q][:n]
            elif op == "trim":
                q = rng.choice(live)
                n = rng.randint(0, len(want[q]))
                m.trim(q, n)
                del want[q][n:]
            else:
                some = rng.sample(live, rng.randint(1, min(3, len(live))))
                m.close(some)
                for q in some:
                    del want[q]
        except Refused as e:
            assert e.args[0] == 2, e.args  # only exhaustion: the arguments were fine
            refused += 1
        held = set()
        for q, rows in want.items():
            length, t = m.table(q)
            assert length == len(rows) and len(t) == -(-length // page)
            assert [int(m.pool[t[i // page], i % page]) for i in range(length)] == rows
            held |= set(t)
        assert m.available() == 40 - len(held)
    assert refused > 0
    lib.pm_delete(m.m)


def test_pages_are_taken_lowest_first(lib):
    m = Map(lib, 8, 4, 4, 32)
    a, b = m.open(), m.open()
    m.extend([a, b], [5, 3])
    assert m.table(a)[1] == [0, 1] and m.table(b)[1] == [2]
    m.close([a])
    m.extend([b], [6])
    assert m.table(b)[1] == [2, 0, 1]


def test_shared_last_page_is_copied_on_growth(lib):
    m = Map(lib, 8, 4, 4, 32)
    a = m.open()
    m.extend([a], [6])
    m.pool[:2] = np.arange(8).reshape(2, 4)
    b, c = m.fork(a, 5, 2)
    assert m.available() == 6
    m.extend([a, b, c], [1, 1, 1])  # two copies; the last holder keeps the page
    assert m.copies[:2].tolist() == [[1, 2, 2], [1, 3, 1]]
    assert m.table(a)[1] == [0, 2] and m.table(b)[1] == [0, 3] and m.table(c)[1] == [0, 1]
    assert m.available() == 4


def test_refusals_change_nothing(lib):
    m = Map(lib, 4, 4, 3, 24)
    a = m.open()
    m.extend([a], [9])
    b = m.fork(a, 9, 1)[0]

    def state():
        return m.available(), m.table(a), m.table(b)

    before = str(state())
    for want, call in [
        (2, lambda: m.extend([a, b], [4, 1])),      # 1 page + a copy + 1 page, one free
        (1, lambda: m.extend([a, a], [1, 1])),      # the same sequence twice
        (1, lambda: m.extend([a], [16])),           # past max_len
        (1, lambda: m.extend([a], [2 ** 64 - 8])),  # a length that wraps
        (1, lambda: m.extend([0], [1])),
        (1, lambda: m.extend([77], [1])),
        (1, lambda: m.fork(a, 10, 1)),
        (2, lambda: m.fork(a, 9, 2)),               # one sequence left
        (2, lambda: m.copy(a, 9)),                  # three pages, one free
        (1, lambda: m.copy(a, 10)),
        (1, lambda: m.trim(a, 10)),
        (1, lambda: m.close([a, a])),
        (1, lambda: m.close([a, 5])),
    ]:
        with pytest.raises(Refused) as e:
            call()
        assert e.value.args[0] == want, e.value.args
        assert str(state()) == before
    m.close([b])
    again = m.open()
    assert again != b
    with pytest.raises(Refused):
        m.trim(b, 0)  # a closed handle stays closed though its place is taken
