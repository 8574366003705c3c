"""The paged cache's bookkeeping when a step or a compaction cannot be enqueued
(kernrt_b200/csrc/pages.cpp, no GPU): a map on which extends are taken back and
compactions only planned stays the same, page for page and in what it hands out
next, as one that never saw them."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

from tests import test_pages
from tests.test_pages import Map, Refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
S = C.c_size_t


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("pages") / "pages.so")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", so,
                    os.path.join(ROOT, "tests", "cpp", "pages_undo_driver.cpp"),
                    os.path.join(ROOT, "kernrt_b200", "csrc", "pages.cpp")], check=True)
    lib = C.CDLL(so)
    U64 = C.c_uint64
    lib.pm_new.restype, lib.pm_new.argtypes = C.c_void_p, [S] * 4
    lib.pm_msg.restype = C.c_char_p
    lib.pm_available.restype = lib.pm_compact.restype = lib.pm_plan_compact.restype = S
    for name, args in (("pm_delete", []), ("pm_available", []), ("pm_open", [C.POINTER(U64)]),
                       ("pm_fork", [U64, S, S, C.c_void_p]), ("pm_copy", [U64, S, C.POINTER(U64), C.c_void_p, C.POINTER(S)]),
                       ("pm_trim", [U64, S]), ("pm_close", [C.c_void_p, S]),
                       ("pm_extend", [C.c_void_p, C.c_void_p, S, C.c_void_p, C.POINTER(S)]),
                       ("pm_compact", [C.c_void_p]), ("pm_plan_compact", [C.c_void_p]),
                       ("pm_undo_extend", [C.c_void_p, C.c_void_p, S, C.c_void_p, S]),
                       ("pm_table", [U64, C.POINTER(S), C.c_void_p, C.POINTER(S), C.POINTER(S)])):
        getattr(lib, name).argtypes = [C.c_void_p] + args
    return lib


def extend_and_undo(m, seqs, rows):
    a, r, n = np.array(seqs, np.uint64), np.array(rows, np.uint64), S()
    m._ok(m.lib.pm_extend(m.m, a.ctypes.data, r.ctypes.data, a.size, m.copies.ctypes.data, C.byref(n)))
    m.lib.pm_undo_extend(m.m, a.ctypes.data, r.ctypes.data, a.size, m.copies.ctypes.data, n.value)
    return n.value


@pytest.mark.parametrize("seed", range(8))
def test_extends_taken_back_leave_no_trace(lib, seed):
    rng = random.Random(seed)
    page = rng.choice([1, 2, 4, 16])
    one, two = (Map(lib, 40, page, 9, 40 * page) for _ in range(2))
    live, copied, undone = {}, 0, 0

    def both(call):
        got = []
        for m in (one, two):
            try:
                got.append(call(m))
            except Refused as e:
                got.append(e.args)
        assert got[0] == got[1]
        return got[0]

    def state(m):
        return m.available(), {q: m.table(q) for q in live}

    for _ in range(800):
        if live:
            some = rng.sample(list(live), rng.randint(1, len(live)))
            rows = [rng.choice([0, 1, 1, 1, 3, page, 5 * page]) for _ in some]
            before = str(state(two))
            try:
                copied += extend_and_undo(two, some, rows)
                undone += 1
            except Refused as e:
                assert e.args[0] == 2
            planned = two.lib.pm_plan_compact(two.m, two.copies.ctypes.data)
            plan = two.copies[:planned].tolist()
            assert str(state(two)) == before
        op = rng.choice(["open", "extend", "extend", "extend", "fork", "fork", "copy", "trim", "close", "compact"])
        q = rng.choice(list(live)) if live else None
        if op == "open":
            h = both(lambda m: m.open())
            if isinstance(h, int):
                live[h] = 0
        elif op == "compact":
            n = both(lambda m: m.compact())
            if live:
                assert n == planned and two.copies[:n].tolist() == plan
        elif q is None:
            continue
        elif op == "extend":
            some = rng.sample(list(live), rng.randint(1, len(live)))
            rows = [rng.choice([0, 1, 1, 3, page]) for _ in some]
            if both(lambda m: m.extend(some, rows)) is None:
                for s, n in zip(some, rows):
                    live[s] += n
        elif op == "fork":
            n, k = rng.randint(0, live[q]), rng.randint(1, 3)
            got = both(lambda m: m.fork(q, n, k))
            if isinstance(got, list):
                live.update((c, n) for c in got)
        elif op == "copy":
            n = rng.randint(0, live[q])
            got = both(lambda m: m.copy(q, n))
            if isinstance(got, int):
                live[got] = n
        elif op == "trim":
            live[q] = rng.randint(0, live[q])
            both(lambda m: m.trim(q, live[q]))
        else:
            both(lambda m: m.close([q]))
            del live[q]
        assert str(state(one)) == str(state(two))
    assert undone > 100 and (copied > 0 or page == 1)  # (a page of one position is never shared in part)
    for m in (one, two):
        lib.pm_delete(m.m)


def test_a_copy_on_write_is_taken_back(lib):
    m = Map(lib, 8, 4, 4, 32)
    a = m.open()
    m.extend([a], [6])
    b, c = m.fork(a, 5, 2)
    before = str((m.available(), m.table(a), m.table(b), m.table(c)))
    assert extend_and_undo(m, [a, b, c], [1, 9, 1]) == 2
    assert str((m.available(), m.table(a), m.table(b), m.table(c))) == before
    m.extend([c, a, b], [1, 1, 1])
    assert m.table(c)[1] == [0, 2] and m.table(a)[1] == [0, 3] and m.table(b)[1] == [0, 1]


def test_the_bookkeeping_tests_hold_with_this_build(lib):
    test_pages.test_refusals_change_nothing(lib)
    test_pages.test_shared_last_page_is_copied_on_growth(lib)
