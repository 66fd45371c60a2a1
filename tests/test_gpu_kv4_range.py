"""Attention over the 4-bit cache where a position far above the others has no part in the
output (an attention sink whose V row is zero), and for queries of any size by every way a
call runs.

The bound stays 2e-5 of a row's largest value.  A weight is held against the largest that its
wavefront has seen, w, as an fp16 pair of w 2^11 whose low half is held 2^11 higher: w >= 2^-25 to
2^-22 of itself, less to 2^-47.  At 20 nats (2^-28.9) that is at most 2^-18 = 3.8e-6 of a weight,
should all of them be off to the same side; the scores' own error at a score S is S 4 2^-24, at
30 7e-6.  Queries: the same, as their size only scales the scores' unit."""
import numpy as np
import pytest

from tests import kv4_ref as ref
from tests.gpu_helpers import dev
from tests.test_gpu_kv4 import Cache, _attention, _close, _want

pytestmark = pytest.mark.gpu


def _sinks(rng, name, nseq, longest, sinks):
    """A cache whose sequences hold a zero V row at positions `sinks`, and queries for it that
    score those `gap` above the others' mean (the others spread by `spread`)."""
    c = Cache(rng, name, nseq, longest, 64)
    n = c.npages * 64
    k = np.zeros((n, c.kv, c.D), np.float32)
    k[:, :, 0] = 8.0  # the first block's scale is 1: dim 1 holds whole numbers
    k[:, :, 32:] = rng.standard_normal((n, c.kv, c.D - 32))
    if c.D == 32:
        k[:, :, 2:] = rng.integers(-1, 2, (n, c.kv, 30))
    v = rng.standard_normal((n, c.kv, c.D)).astype(np.float32)
    for pages in c.pages:
        for p in sinks:
            row = pages[p // 64] * 64 + p % 64
            k[row, :, 1:] = 0
            k[row, :, 1] = 7
            v[row] = 0
    c.k0, c.v0 = ref.pack(k, c.kv, c.D, 64, True), ref.pack(v, c.kv, c.D, 64, False)
    c.k, c.v = dev(c.k0), dev(c.v0)

    def queries(nq, gap, spread):
        q = rng.standard_normal((nq, c.q, c.D)).astype(np.float32) * spread
        q[:, :, 0] = 0
        q[:, :, 1] = gap * np.sqrt(c.D) / 7
        return q
    return c, queries


GAPS = [(10, 0.3), (14, 0.3), (17, 0.0), (20, 0.0), (20, 0.3)]


@pytest.mark.parametrize("name,nq,n", [
    ("g7_d128", 1, 512), ("g7_d128", 16, 1500), ("g7_d128", 1, 5000), ("g7_d128", 200, 260),
    ("g7_d64", 3, 1100), ("g1_d32", 1, 3000), ("g3_d96", 4, 700),
    ("g16_d64", 1, 500), ("g16_d64", 2, 4000), ("g9_d32", 30, 900), ("g16_d128", 5, 2500)])
def test_sinks_of_queries(name, nq, n):
    """One query a sequence: whole contexts in four and in eight wavefronts, and split."""
    rng = np.random.default_rng(n + nq)
    c, queries = _sinks(rng, name, nq, n, [3])
    some = sorted({0, nq // 2, nq - 1})
    ctx = dev(np.full(nq, n, np.int32))
    for gap, spread in GAPS:
        q = queries(nq, gap, spread)
        want = _want(c, q[some], some, [n] * len(some))
        _close(_attention(c, dev(q), nq, None, n, 0, n)[some], want, (gap, "host contexts"))
        _close(_attention(c, dev(q), nq, ctx, 0, 0, n)[some], want, (gap, "device contexts"))


@pytest.mark.parametrize("name,nq,first", [
    ("g7_d128", 2, 700), ("g7_d128", 20, 1500), ("g16_d64", 40, 300), ("g9_d32", 3, 4000),
    ("g1_d32", 60, 900), ("g3_d96", 33, 600),
    # by fp16 rows: every kernel that takes them
    ("g7_d128", 322, 700), ("g7_d128", 1500, 100), ("g7_d64", 700, 500), ("g16_d64", 1030, 64),
    ("g3_d96", 400, 900), ("g3_d96", 1000, 50), ("g3_d96", 1800, 50), ("g1_d32", 1200, 300),
    ("g1_d32", 4100, 100)])
def test_sinks_of_prompts(name, nq, first):
    rng = np.random.default_rng(first + nq)
    c, queries = _sinks(rng, name, 1, first + nq, [0, 37])
    some = sorted({0, 1, nq // 2, nq - 1})
    for gap, spread in GAPS:
        q = queries(nq, gap, spread)
        got = _attention(c, dev(q), nq, None, first + 1, 1, first + nq)
        _close(got[some], _want(c, q[some], [0] * len(some), first + 1 + np.array(some)), gap)


@pytest.mark.parametrize("name,nq,first", [("g7_d128", 322, 40), ("g7_d128", 1470, 0),
                                           ("g16_d128", 600, 30), ("g7_d64", 650, 9),
                                           ("g3_d96", 380, 70), ("g1_d32", 1130, 33)])
@pytest.mark.parametrize("size", [1e30, 1e38, 3.4e38, 7e4, 1e-6, 1e-38])
def test_queries_of_any_size_by_rows(name, nq, first, size):
    """Prompts of more than 9000 (query, head) rows.  1e30 and more: every weight 0 or 1 (the two
    best of some hundred scores differ by far more than a rounding of either).  The others, 7e4
    just past fp16's largest, over K of a size that makes ordinary scores of them (1e-38: none):
    weights that differ in their bits."""
    rng = np.random.default_rng(nq)
    c = Cache(rng, name, 1, first + nq, 32)
    some = np.array(sorted({0, 1, nq // 3, nq - 2, nq - 1}))
    if size < 1e5:
        x = rng.standard_normal((c.npages * 32, c.kv, c.D)).astype(np.float32)
        x *= np.float32(1e-4 if size > 1 else 2e4)
        c.k0 = ref.pack(x, c.kv, c.D, 32, True)
        c.k = dev(c.k0)
    q = (np.clip(rng.standard_normal((nq, c.q, c.D)), -1, 1) * size).astype(np.float32)
    got = _attention(c, dev(q), nq, None, first + 1, 1, first + nq)
    _close(got[some], _want(c, q[some], [0] * len(some), first + 1 + some), (name, size))
    # beside rows of other sizes, and of NaN, in the same tile: the same bits
    q2 = q.copy()
    q2[some[2], 0], q2[some[2], 1] = np.nan, 1.0
    again = _attention(c, dev(q2), nq, None, first + 1, 1, first + nq, q8=False)
    keep = np.ones((nq, c.q), bool)
    keep[some[2], :2] = False
    assert np.array_equal(got[keep], again[keep])
    assert np.isnan(again[some[2], 0]).all() and np.isfinite(again[some[2], 1]).all()


@pytest.mark.parametrize("name,nq", [("g7_d128", 1), ("g9_d32", 1), ("g7_d128", 5), ("g7_d64", 700)])
def test_scores_at_the_end_of_fp32(name, nq):
    """A maximum whose last place is about a weight's range: no weight past fp16's largest."""
    rng = np.random.default_rng(nq)
    n = 800
    c = Cache(rng, name, 1, n, 64)
    x = np.zeros((c.npages * 64, c.kv, c.D), np.float32)
    x[:, :, 0] = 8.0
    x[:, :, 1:] = rng.integers(-4, 5, (len(x), c.kv, c.D - 1))
    c.k0 = ref.pack(x, c.kv, c.D, 64, True)
    c.k = dev(c.k0)
    v = np.abs(c.rows(c.v0, 0, np.arange(n), False)).max()
    for e in range(16, 40):
        q = rng.integers(-8, 9, (nq, c.q, c.D)).astype(np.float32)
        q[:, :, 0] = 2.0 ** e
        got = _attention(c, dev(q), nq, None, n - nq + 1, 1 if nq > 1 else 0, n)
        # (a mean of V rows, but for the weights' own rounding)
        assert np.isfinite(got).all() and np.abs(got).max() <= v * 1.0001, e
