"""Bookkeeping of lengths up to an int's largest, and of compactions whose copies are pending
(libsi_host.so, on the CPU)."""
import ctypes

import numpy as np
import pytest

import si_amd
from tests.test_kvpages_share import PS, Pool


@pytest.fixture
def H():
    return si_amd.host_lib()


@pytest.mark.parametrize("page_size", [1 << 16, 1 << 30])
def test_lengths_up_to_the_largest(H, page_size):
    """A length within a page of 2^31: forks share every page, and truncation keeps them."""
    top = 2 ** 31 - 1
    need = -(-top // page_size)
    p = H.si_kv_pages_create(need + 1, page_size, 3, need)
    try:
        a = H.si_kv_seq_add(p)
        assert H.si_kv_seq_grow(p, a, top) == 0 and H.si_kv_pages_free(p) == 1
        b = H.si_kv_seq_fork(p, a)
        table = np.ctypeslib.as_array(H.si_kv_page_table(p), shape=(3, need))
        assert H.si_kv_seq_len(p, b) == top and np.array_equal(table[a], table[b])
        H.si_kv_seq_truncate(p, a, top - 1)
        H.si_kv_seq_truncate(p, b, top - 1)
        assert H.si_kv_pages_free(p) == 1 and np.array_equal(table[a], np.arange(need))
        H.si_kv_seq_free(p, a)
        assert H.si_kv_pages_free(p) == 1  # b holds them still
        H.si_kv_seq_truncate(p, b, page_size)
        assert H.si_kv_pages_free(p) == need
    finally:
        H.si_kv_pages_destroy(p)


def test_compaction_counts_the_pages_it_moves(H):
    """Held pages are what compaction returns, with its copies pending and after them: a moved
    page counts once more until its copy is done."""
    rng = np.random.default_rng(4)
    p = Pool(H, 40)
    try:
        for turn in range(40):
            seqs = [s for s in (p.add() for _ in range(3)) if s >= 0]
            for s in seqs:
                p.grow(s, int(rng.integers(1, 30)))
            p.step()
            for s in rng.permutation(list(p.want))[:2]:
                p.free(int(s))
            p.step()
            used = H.si_kv_compact(p.p)
            assert used == p.npages - H.si_kv_pages_free(p.p) - len(p.copies()[0])
            p.step()
            assert used == p.npages - H.si_kv_pages_free(p.p)
            held = {int(x) for s, t in p.want.items() for x in p.table(s)[:-(-len(t) // PS)]}
            assert held == set(range(used))
    finally:
        p.close()
