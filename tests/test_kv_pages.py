"""The page books of a paged cache (who holds which page, what is copied) against a model that keeps every sequence's
positions as a list: random calls, refusals, and that a refused call changes nothing.  No GPU: the header is host code."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
FULL, INVALID = -2, -3


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv_pages") / "kv_pages_host.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-Wall", "-Werror", "-shared", "-fPIC",
                    os.path.join(HERE, "kv_pages_host.cpp"), "-o", so], check=True)
    h = ctypes.CDLL(so)
    h.kv_new.restype, h.kv_why.restype = ctypes.c_void_p, ctypes.c_char_p
    return h


class Books:
    def __init__(self, lib, page, n_pages, max_seqs, max_pages):
        self.lib, self.page, self.n_pages, self.max_seqs, self.max_pages = lib, page, n_pages, max_seqs, max_pages
        self.c = ctypes.c_void_p(lib.kv_new(page, n_pages, max_seqs, max_pages))

    @staticmethod
    def _u32(v):
        return np.ascontiguousarray(v, np.uint32)

    def extend(self, seqs, n):
        s, n = self._u32(seqs), self._u32(n)
        return self.lib.kv_extend(self.c, len(s), s.ctypes.data_as(ctypes.c_void_p), n.ctypes.data_as(ctypes.c_void_p))

    def truncate(self, seqs, n):
        s, n = self._u32(seqs), self._u32(n)
        return self.lib.kv_truncate(self.c, len(s), s.ctypes.data_as(ctypes.c_void_p), n.ctypes.data_as(ctypes.c_void_p))

    def fork(self, src, dsts, n):
        d = self._u32(dsts)
        return self.lib.kv_fork(self.c, ctypes.c_uint32(src), len(d), d.ctypes.data_as(ctypes.c_void_p), ctypes.c_uint32(n))

    def compact(self):
        live = ctypes.c_uint32(99)
        return self.lib.kv_compact(self.c, ctypes.byref(live)), live.value

    def why(self):
        return self.lib.kv_why(self.c).decode()

    def read(self):
        tab, seq = (self.max_seqs, self.max_pages), (self.max_seqs,)
        out = [np.empty(s, np.int32) for s in (tab, seq, seq)] + [ctypes.c_uint32(0)] + \
            [np.empty(s, np.int32) for s in ((self.n_pages, self.page), tab, seq, seq)]
        self.lib.kv_read(self.c, *[ctypes.byref(o) if isinstance(o, ctypes.c_uint32) else o.ctypes.data_as(ctypes.c_void_p) for o in out])
        return [o.value if isinstance(o, ctypes.c_uint32) else o for o in out]


def _holds(b, want):
    """The books agree with the arrays, and the arrays hold the wanted positions."""
    table, lens, own, n_free, pool, d_table, d_lens, d_own = b.read()
    assert np.array_equal(table, d_table) and np.array_equal(lens, d_lens) and np.array_equal(own, d_own)
    used = set()
    for s, values in enumerate(want):
        assert lens[s] == len(values) and 0 <= own[s] <= len(values)
        need = -(-len(values) // b.page)
        assert (table[s, need:] == -1).all() and (table[s, :need] >= 0).all()
        used |= set(table[s, :need].tolist())
        got = pool[table[s, :need]].reshape(-1)[:len(values)]
        assert got.tolist() == values, (s, got.tolist(), values)
    assert n_free == b.n_pages - len(used) and b.lib.kv_longest(b.c) == max(len(v) for v in want)
    return table, lens, own, n_free, pool


@pytest.mark.parametrize("page,n_pages,max_seqs,max_pages,seed", [(4, 24, 6, 8, 0), (1, 30, 5, 12, 1), (7, 12, 4, 5, 2), (64, 40, 9, 6, 3), (5, 9, 12, 9, 4)])
def test_random_calls(lib, page, n_pages, max_seqs, max_pages, seed):
    rng = np.random.default_rng(seed)
    b, want, mark, refused, copied = Books(lib, page, n_pages, max_seqs, max_pages), [[] for _ in range(max_seqs)], 0, 0, 0
    for _ in range(1500):
        before = b.read()
        op = rng.choice(["extend", "fork", "truncate", "compact"], p=[0.5, 0.2, 0.25, 0.05])
        seqs = rng.permutation(max_seqs)[:rng.integers(1, max_seqs + 1)]
        if op == "extend":
            n = rng.integers(0, 2 * page + 2, len(seqs))
            rc = b.extend(seqs, n)
            if rc == 0:
                for s, k in zip(seqs, n):
                    for p in range(len(want[s]), len(want[s]) + k):
                        mark += 1
                        want[s].append(mark)
                        assert lib.kv_write(b.c, int(s), int(p), mark) == 0
        elif op == "fork":
            src, dsts = int(seqs[0]), [int(d) for d in seqs[1:] if rng.random() < 0.9 and not want[d]]
            n = int(rng.integers(0, len(want[src]) + 1))
            rc = b.fork(src, dsts, n)
            assert rc == 0
            for d in dsts:
                want[d] = want[src][:n]
        elif op == "truncate":
            to = [int(rng.integers(0, len(want[s]) + 1)) if rng.random() < 0.6 else 0 for s in seqs]
            rc = b.truncate(seqs, to)
            assert rc == 0
            for s, k in zip(seqs, to):
                want[s] = want[s][:k]
        else:
            rc, live = b.compact()
            assert rc == 0
            table = b.read()[0]
            assert live == len(set(table[table >= 0].tolist())) and (live == 0 or table.max() == live - 1)
        if rc:
            refused += 1
            after = b.read()
            assert all(np.array_equal(x, y) for x, y in zip(before, after)) and b.why()
        table, lens, own, _, _ = _holds(b, want)
        # a position that two sequences hold is nobody's to write
        for s in range(max_seqs):
            for t in range(s):
                m = min(len(want[s]), len(want[t]))
                both = np.flatnonzero(table[s, :-(-m // page)] == table[t, :-(-m // page)]) if m else []
                for j in both:
                    shared = [p for p in range(j * page, min(m, (j + 1) * page)) if want[s][p] == want[t][p]]
                    assert all(p < own[s] and p < own[t] for p in shared)
                    copied += len(shared)
    assert refused > 20 and copied > 100
    lib.kv_delete(b.c)


def test_last_holder_keeps_the_page(lib):
    b = Books(lib, 4, 10, 4, 3)
    assert b.extend([0], [6]) == 0 and b.fork(0, [1, 2], 6) == 0
    assert b.extend([0, 1, 2], [1, 1, 1]) == 0
    table = b.read()[0]
    assert table[:3, :2].tolist() == [[0, 2], [0, 3], [0, 1]] and b.read()[3] == 6
    lib.kv_delete(b.c)
    # room is counted with the copies: the last of three holders needs none
    b = Books(lib, 4, 3, 4, 3)
    assert b.extend([0], [5]) == 0 and b.fork(0, [1, 2], 5) == 0
    before = b.read()
    assert b.extend([0, 1, 2], [1, 1, 1]) == FULL and "2 pages needed, 1 of 3 free" in b.why()
    assert all(np.array_equal(x, y) for x, y in zip(before, b.read()))
    assert b.truncate([2], [0]) == 0 and b.extend([0, 1], [1, 1]) == 0 and b.read()[3] == 0
    lib.kv_delete(b.c)


def test_lowest_free_page_first_and_compaction_in_order(lib):
    b = Books(lib, 2, 8, 4, 4)
    assert b.extend([0, 1, 2], [4, 4, 4]) == 0 and b.truncate([0], [0]) == 0
    assert b.extend([3], [2]) == 0
    assert b.read()[0][3, 0] == 0
    assert b.truncate([3], [0]) == 0 and b.compact() == (0, 4)
    assert b.read()[0][1:3, :2].tolist() == [[2, 3], [0, 1]]
    lib.kv_delete(b.c)


def test_refusals(lib):
    b = Books(lib, 4, 8, 3, 2)
    assert b.extend([0], [3]) == 0
    before = b.read()
    for call, text in [(lambda: b.extend([3], [1]), "sequence 3"), (lambda: b.extend([0, 0], [1, 1]), "twice"), (lambda: b.extend([0], [6]), "at most 8"),
                       (lambda: b.extend([1], [0xFFFFFFFF]), "at most 8"), (lambda: b.fork(0, [0], 1), "not empty"), (lambda: b.fork(3, [1], 0), "sequence 3"),
                       (lambda: b.fork(0, [1], 4), "4 positions"), (lambda: b.fork(1, [0], 0), "not empty"), (lambda: b.truncate([0], [4]), "to 4"),
                       (lambda: b.truncate([0, 0], [1, 1]), "twice"), (lambda: b.truncate([9], [0]), "sequence 9")]:
        assert call() == INVALID and text in b.why(), text
    assert b.lib.kv_extend(b.c, 1, None, None) == INVALID and "null" in b.why()
    assert b.extend([0], [6]) == INVALID and "at most 8" in b.why()
    assert b.extend([], []) == 0 and b.fork(0, [], 2) == 0 and b.extend([1], [0]) == 0
    assert all(np.array_equal(x, y) for x, y in zip(before, b.read()))
    lib.kv_delete(b.c)
