"""Prompts so long that four 32-row tiles share a workgroup (k_attn_rows<D, 4, ...>): head dims,
page sizes, several sequences, Q8_0 outputs, and what their rows do not see.  Each test looks at
which kernel ran, so that it keeps reaching the one that it is for."""
import numpy as np
import pytest

import si_amd
from tests.gpu_helpers import torch_cuda
from tests.test_gpu_step import P, Batch, host, st
from tests.test_gpu_step_values import attend, put

pytestmark = pytest.mark.gpu

# heads, and the fewest rows of a call whose 32-row tiles reach 1800 (3500 up to 64 values a head)
FORMS = [((8, 8, 32), 13985), ((14, 2, 64), 7996), ((24, 8, 96), 2390), ((28, 4, 128), 2053),
         ((16, 1, 128), 3599)]


def rows_of(n):
    """(contexts, new rows) of sequences that bring n rows: a long piece, single tokens, drafts, a
    piece from the start, one without rows, one of a row more than whole tiles."""
    new = [1, n // 5, 0, 6, 129, 1]
    ctx = [400, n // 5, 70, 333, 200, 1]
    new.append(n - sum(new))
    ctx.append(new[-1] + 77)
    return ctx, new


def row_tiles(b, call):
    """Runs call, and gives the row tiles a workgroup of the attention kernel that ran."""
    names = [n for n, _ in si_amd.kernel_times_ms("k_attn_rows<", call)]
    assert len(names) == 1, names
    dim, tiles = names[0].split("<")[1].split(",")[:2]
    assert int(dim) == b.heads[2]
    return int(tiles)


def ran(b):
    """A batch's outputs, and the row tiles a workgroup."""
    got = []
    tiles = row_tiles(b, lambda: got.append(b.run()))
    return got[0], tiles


@pytest.mark.parametrize("heads,least", FORMS)
@pytest.mark.parametrize("page,window,sinks", [(8, 150, 4), (16, 90, 40), (64, 200, 0),
                                               (16, 1, 0), (128, 40, 3)])
def test_prompts(heads, least, page, window, sinks):
    """At the fewest rows of this form, and with room behind them."""
    ctx, new = rows_of(least - 5)
    b = Batch(heads, ctx, new, page, window, sinks, seed=page, room=5)
    got, tiles = ran(b)
    assert tiles == 4
    b.check(got, every=211)


@pytest.mark.parametrize("heads,least", FORMS)
def test_prompts_one_row_fewer(heads, least):
    """The largest calls of the other form."""
    ctx, new = rows_of(least - 1)
    b = Batch(heads, ctx, new, 32, 120, 4, seed=1)
    got, tiles = ran(b)
    assert tiles == 1
    b.check(got, every=211)


@pytest.mark.parametrize("heads,least", FORMS)
@pytest.mark.parametrize("page", [4, 16, 256])
def test_prompts_one_sequence(heads, least, page):
    """One prompt from its start, seeing all of it or a window."""
    for window, sinks in ((2 ** 31 - 1, 0), (700, 70)):
        b = Batch(heads, [least], [least], page, window, sinks, seed=page)
        got, tiles = ran(b)
        assert tiles == 4
        b.check(got, every=1013)


@pytest.mark.parametrize("heads,least", FORMS)
def test_prompts_quantized(heads, least):
    """Outputs and their Q8_0 (with and without block sums), as si_quantize_q8_rows has it; rows
    behind the last are left as they were."""
    torch = torch_cuda()
    ctx, new = rows_of(least)
    b = Batch(heads, ctx, new, 16, 100, 4, room=3).upload()
    n, qd = b.max_rows, heads[0] * heads[2]
    bufs = [[torch.full((n, qd), 7.0, device="cuda"),
             torch.full((n, qd), 7, dtype=torch.int8, device="cuda"),
             torch.full((n, qd // 32), 7, dtype=torch.int16, device="cuda"),
             torch.full((n, qd // 32), 7, dtype=torch.int16, device="cuda")] for _ in range(2)]
    assert row_tiles(b, lambda: b.call(bufs[0][0], bufs[0][1:])) == 4
    b.call(bufs[1][0], (bufs[1][1], bufs[1][2], None))
    qs, d, s = (torch.empty_like(x) for x in bufs[0][1:])
    si_amd.call("si_quantize_q8_rows", P(bufs[0][0]), n, qd, P(qs), P(d), P(s), st())
    for got, want in zip(bufs[0][1:], (qs, d, s)):
        assert torch.equal(got[:b.rows], want[:b.rows])
        assert (got[b.rows:] == 7).all()
    for x, y in zip(bufs[0][:3], bufs[1][:3]):
        assert torch.equal(x, y)
    assert (bufs[1][3] == 7).all()
    b.check(host(bufs[0][0]).reshape(n, *heads[::2]), every=1013)


@pytest.mark.parametrize("heads,least", FORMS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_prompts_hidden_values(heads, least, bad):
    """What a row does not see has no influence on it, in whichever of a workgroup's four row tiles
    it is: bad keys and values at a position that some of its rows see."""
    window, sinks = 90, 4
    b = Batch(heads, [least + 300], [least], 16, window, sinks, seed=3, garbage=bad)
    clean, tiles = ran(b)
    assert tiles == 4
    b.check(clean, every=1013)
    first = 300  # position of the first row
    for at in (first + least - 1, first - window + 1, first + least // 2, first + 130):
        k, v = (x.copy() for x in (b.kpool, b.vpool))
        slot = b.pages[0, at // 16], at % 16
        b.kpool[slot], b.vpool[slot] = bad, bad
        got = b.run()
        p = first + np.arange(least)
        sees = (p >= at) & (p - window < at)
        assert 0 < sees.sum() <= window
        assert np.array_equal(got[~sees], clean[~sees]), at
        assert not np.isfinite(got[sees]).any()
        b.kpool, b.vpool = k, v


@pytest.mark.parametrize("heads,least", FORMS)
@pytest.mark.parametrize("page", [8, 16, 64])
def test_prompts_values_that_are_seen(heads, least, page):
    """Infinities and NaN that some rows of a workgroup's four tiles see, in whole and cut tiles of
    theirs: the definition's outputs there, every other row as it is without them."""
    window, sinks, first = 200, 4, 300
    b = Batch(heads, [least + first], [least], page, window, sinks, seed=page)
    clean, tiles = ran(b)
    assert tiles == 4
    sees = np.zeros(least, bool)
    p = first + np.arange(least)
    bad = [(first - window + 1, "v", np.inf), (first + 40, "k", np.inf), (first + 500, "v", np.nan),
           (first + 777, "v", -np.inf), (first + least // 2, "k", np.nan),
           (first + least - 90, "v", np.inf), (first + least - 1, "v", -np.inf)]
    for n, (at, what, value) in enumerate(bad):
        put(b, 0, at, n % heads[1], 5 * n, **{what: value})
        sees |= (p >= at) & (p - window < at)
    got = b.run()
    assert np.array_equal(got[~sees], clean[~sees])
    edges = [at + d - first for at, _, _ in bad for d in (0, 1, 31, 32, 100, window - 1, window)]
    for j in sorted({j for j in edges if 0 <= j < least}):
        want, bound = attend(b.q[j], b.k[0], b.v[0], first + j, window, sinks,
                             heads[0] // heads[1])
        fine = np.isfinite(want)
        assert np.array_equal(got[j][~fine], want[~fine], equal_nan=True), j
        assert (np.abs(got[j][fine] - want[fine]) <= bound[fine]).all(), j


def test_prompts_repeat():
    """The same bits from call to call."""
    heads, least = FORMS[3]
    ctx, new = rows_of(least + 900)
    b = Batch(heads, ctx, new, 64, 500, 4)
    first, tiles = ran(b)
    assert tiles == 4
    for _ in range(3):
        assert np.array_equal(b.run(), first)
