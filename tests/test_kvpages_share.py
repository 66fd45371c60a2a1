"""Sequences that share pages (si_kv_seq_fork, _truncate, si_kv_copies, si_kv_compact,
si_kv_pages_resize; libsi_host.so) on the CPU, against what they are for: a pool of
pages as a program keeps it, whose copies run when the bookkeeping says.  Every
sequence then reads the positions it was given, whatever the others do."""
import ctypes

import numpy as np
import pytest

import si_amd

PS, MAXP, SEQS = 8, 12, 7


@pytest.fixture
def H():
    return si_amd.host_lib()


class Pool:
    """Pages of position tags; each sequence's own tags beside them."""

    def __init__(self, H, npages):
        self.H, self.npages = H, npages
        self.p = H.si_kv_pages_create(npages, PS, SEQS, MAXP)
        self.mem = np.full((npages, PS), -1, np.int64)
        self.want = {}
        self.tag = 0

    def table(self, seq):
        t = np.ctypeslib.as_array(self.H.si_kv_page_table(self.p), shape=(SEQS * MAXP,))
        return t.reshape(SEQS, MAXP)[seq]

    def copies(self):
        P = ctypes.POINTER(ctypes.c_int)
        src, dst = P(), P()
        n = self.H.si_kv_copies(self.p, ctypes.byref(src), ctypes.byref(dst))
        return src[:n], dst[:n]

    def run_copies(self):
        src, dst = self.copies()
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)  # they run at once
        assert all(0 <= x < self.npages for x in src + dst)
        self.mem[dst] = self.mem[src]
        self.H.si_kv_copies_done(self.p)
        assert self.copies() == ([], [])

    def add(self):
        s = self.H.si_kv_seq_add(self.p)
        if s >= 0:
            self.want[s] = []
        return s

    def grow(self, seq, by):
        n = len(self.want[seq])
        if self.H.si_kv_seq_grow(self.p, seq, n + by) != 0:
            return False
        self.new = getattr(self, "new", [])
        self.new += [(seq, i) for i in range(n, n + by)]
        self.want[seq] += [None] * by
        return True

    def step(self):
        """Copies, then the new positions are written (a decode step's append)."""
        self.run_copies()
        for seq, i in getattr(self, "new", []):
            if seq in self.want and i < len(self.want[seq]) and self.want[seq][i] is None:
                self.tag += 1
                self.mem[self.table(seq)[i // PS], i % PS] = self.tag
                self.want[seq][i] = self.tag
        self.new = []
        self.check()

    def fork(self, seq):
        s = self.H.si_kv_seq_fork(self.p, seq)
        if s >= 0:
            self.want[s] = list(self.want[seq])
        return s

    def truncate(self, seq, n):
        self.H.si_kv_seq_truncate(self.p, seq, n)
        del self.want[seq][n:]

    def free(self, seq):
        self.H.si_kv_seq_free(self.p, seq)
        del self.want[seq]

    def check(self):
        held = set()
        for seq, tags in self.want.items():
            assert self.H.si_kv_seq_len(self.p, seq) == len(tags)
            t = self.table(seq)
            got = [self.mem[t[i // PS], i % PS] for i in range(len(tags))]
            assert got == tags, seq
            held |= {int(t[i]) for i in range(-(-len(tags) // PS))}
        if self.copies() == ([], []):
            assert self.H.si_kv_pages_free(self.p) == self.npages - len(held)

    def close(self):
        self.H.si_kv_pages_destroy(self.p)


def test_fork_shares_and_copies_once(H):
    p = Pool(H, 6)
    try:
        a = p.add()
        assert p.grow(a, 20)  # pages 0, 1, 2; the last holds 4 positions
        p.step()
        b = p.fork(a)
        assert H.si_kv_pages_free(p.p) == 3 and list(p.table(b)[:3]) == [0, 1, 2]
        assert p.copies() == ([], [])
        # the first to grow gets a page of its own, the other keeps the old one
        assert p.grow(b, 1) and p.copies() == ([2], [3])
        assert p.grow(a, 1) and p.copies() == ([2], [3])
        assert H.si_kv_pages_free(p.p) == 2
        p.step()
        assert list(p.table(a)[:3]) == [0, 1, 2] and list(p.table(b)[:3]) == [0, 1, 3]
        # whole pages are shared without a copy
        p.truncate(b, 16)
        c = p.fork(b)
        assert p.grow(c, 3) and p.copies() == ([], [])
        p.step()
        p.free(a)
        p.step()
        assert H.si_kv_pages_free(p.p) == 3  # 0 and 1 are b's and c's still
    finally:
        p.close()


def test_copy_of_a_pending_copy(H):
    """A fork of a sequence whose page is still to be copied reads what that copy reads."""
    p = Pool(H, 8)
    try:
        a = p.add()
        assert p.grow(a, 5)
        p.step()
        b = p.fork(a)
        assert p.grow(b, 0) and p.copies() == ([], [])  # nothing is written
        assert p.grow(b, 1) and p.copies() == ([0], [1])
        c = H.si_kv_seq_fork(p.p, b)  # with b's new position, not written yet
        H.si_kv_seq_truncate(p.p, c, 5)
        p.want[c] = list(p.want[a])
        assert p.grow(c, 2)
        assert p.copies() == ([0, 0], [1, 2])
        p.free(b)  # its copy is dropped, its page free
        assert p.copies() == ([0], [2]) and H.si_kv_pages_free(p.p) == 6
        p.free(a)  # page 0 is held by the copy
        assert H.si_kv_pages_free(p.p) == 6
        p.step()
        assert H.si_kv_pages_free(p.p) == 7
    finally:
        p.close()


def test_exhaustion_counts_the_copy(H):
    p = Pool(H, 3)
    try:
        a = p.add()
        assert p.grow(a, 12)
        p.step()
        b = p.fork(a)
        assert H.si_kv_seq_grow(p.p, b, 12 + 5) == -1  # a copy and a page: one is free
        assert p.copies() == ([], []) and list(p.table(b)[:2]) == [0, 1]
        assert p.grow(b, 4)
        p.step()
        assert H.si_kv_pages_free(p.p) == 0
        assert p.grow(a, 4)  # its page is its own again
        p.step()
    finally:
        p.close()


def test_compact_and_resize(H):
    p = Pool(H, 12)
    try:
        s = [p.add() for _ in range(4)]
        for x in s:
            assert p.grow(x, 20)
        p.step()
        f = p.fork(s[3])
        p.free(s[0])
        p.free(s[2])
        p.step()
        assert H.si_kv_pages_resize(p.p, 6) == -1
        assert H.si_kv_compact(p.p) == 6
        src, dst = p.copies()
        assert sorted(dst) == [0, 1, 2] and sorted(src) == [9, 10, 11]
        assert H.si_kv_pages_resize(p.p, 6) == -1  # still read by the copies
        g = p.fork(f)
        assert p.grow(g, 1)  # of a page that is about to move
        p.step()
        assert H.si_kv_pages_resize(p.p, 7) == 0 and H.si_kv_pages_free(p.p) == 0
        p.npages = 7
        p.check()
        assert not p.grow(s[1], 8)
        assert H.si_kv_pages_resize(p.p, 9) == 0
        p.npages, p.mem = 9, np.concatenate([p.mem[:7], np.full((2, PS), -1, np.int64)])
        assert p.grow(s[1], 8) and max(p.table(s[1])[:4]) == 7  # lowest id first
        p.step()
        assert H.si_kv_compact(p.p) == 8 and p.copies() == ([], [])
    finally:
        p.close()


@pytest.mark.parametrize("seed", range(6))
def test_random_workload_keeps_every_sequence(H, seed):
    rng = np.random.default_rng(seed)
    p = Pool(H, 30 + 5 * seed)
    try:
        for _ in range(1500):
            op = rng.integers(0, 12)
            live = list(p.want)
            if op == 0:
                p.add()
            elif not live:
                continue
            else:
                seq = int(rng.choice(live))
                n = len(p.want[seq])
                if op == 1 and None not in p.want[seq]:
                    p.fork(seq)
                elif op == 2:
                    p.free(seq)
                elif op == 3:
                    p.truncate(seq, int(rng.integers(0, n + 1)))
                elif op == 4:
                    p.step()
                    if rng.integers(0, 4) == 0:
                        used = H.si_kv_compact(p.p)
                        assert used == p.npages - H.si_kv_pages_free(p.p) - len(p.copies()[0]) \
                            or p.copies() != ([], [])
                        p.step()
                        tops = [p.table(s)[:-(-len(t) // PS)] for s, t in p.want.items()]
                        assert not tops or max([-1] + [int(x) for t in tops for x in t]) < used
                elif n < MAXP * PS - 20:
                    p.grow(seq, int(rng.integers(0, 20)))
            if rng.integers(0, 3) == 0:
                p.step()
        p.step()
    finally:
        p.close()


@pytest.mark.parametrize("code,msg", [
    ("H.si_kv_seq_fork(p, 1)", "unknown sequence"), ("H.si_kv_seq_truncate(p, 0, 6)", "length"),
    ("H.si_kv_seq_truncate(p, 0, -1)", "length"), ("H.si_kv_pages_resize(p, 0)", "npages"),
    ("H.si_kv_seq_fork(p, 0); H.si_kv_seq_grow(p, 1, 6); H.si_kv_compact(p)", "pending"),
    ("H.si_stack_create_kv(si_amd.make_shape(**si_amd.SHAPES['0.5b']), None, 1, 1, 64, 4, 16, 2)",
     "unknown K/V format"),
    ("H.si_stack_create_kv(si_amd.make_shape(**si_amd.SHAPES['0.5b']), None, 1, 1, 64, 4, 8, 1)",
     "16..65536"),
    ("H.si_stack_create_kv(si_amd.make_shape(896, 14, 2, 48), None, 1, 1, 64, 4, 16, 1)",
     "16..65536")])
def test_misuse_dies(code, msg):
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", "import sys; sys.path[:0] = %r; import si_amd\n"
                        "H = si_amd.host_lib()\np = H.si_kv_pages_create(4, 8, 3, 4)\n"
                        "H.si_kv_seq_add(p); H.si_kv_seq_grow(p, 0, 5)\n%s" % (sys.path, code)],
                       capture_output=True, text=True)
    assert r.returncode == 1 and msg in r.stderr
