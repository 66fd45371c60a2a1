"""Infinities and NaN that a row of si_attention_rows sees: the outputs that the definition gives,
wherever the position lies in the walk and however the walk is cut."""
import numpy as np
import pytest

from tests import step_ref
from tests.test_gpu_step import Batch

pytestmark = pytest.mark.gpu

INF, NAN = np.inf, np.nan


def attend(q, k, v, p, window, sinks, per):
    """(out, bound) as step_ref.attend has them, where k and v may be infinite or NaN: a score of
    NaN or +inf makes the head's outputs NaN, as do scores of -inf alone; an infinite value (or
    NaN) is met by its sign, as NaN where the score is -inf (weight 0)."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    t = step_ref.visible(p, window, sinks)
    for h in range(q.shape[0]):
        kk, vv = k[t, h // per], v[t, h // per]
        with np.errstate(invalid="ignore"):
            s = kk.astype(np.float64) @ q[h].astype(np.float64)
        live = s > -INF
        if np.isnan(s).any() or (s == INF).any() or not live.any():
            out[h] = NAN
            continue
        # (what has no weight says nothing of the others' sums)
        fine = np.where(np.isfinite(vv), vv, 0).astype(np.float16)
        o, b = step_ref.attend(q[h:h + 1], kk[live][:, None], fine[live][:, None],
                               int(live.sum()) - 1, 2 ** 31 - 1, 0, 1)
        met = np.where(np.isfinite(vv), 0.0, np.where(live[:, None], vv.astype(np.float64), NAN))
        with np.errstate(invalid="ignore"):
            out[h], bound[h] = o[0] + met.sum(0), b[0]
    return out, bound


def put(b, i, pos, heads, dims, k=None, v=None):
    """Values at a position of sequence i, in the pools and in the lists."""
    slot = b.pages[i, pos // b.page], pos % b.page
    for x, pool, value in ((b.k, b.kpool, k), (b.v, b.vpool, v)):
        if value is not None:
            x[i][pos][heads, dims] = value
            pool[slot][heads, dims] = value


def check(b, got):
    """Every row's finite outputs within the bound, the others the definition's."""
    for i in range(len(b.ctx)):
        for j in range(int(b.new[i])):
            r = int(b.start[i]) + j
            want, bound = attend(b.q[r], b.k[i], b.v[i], int(b.ctx[i] - b.new[i]) + j, b.window,
                                 b.sinks, b.heads[0] // b.heads[1])
            fine = np.isfinite(want)
            assert np.array_equal(got[r][~fine], want[~fine], equal_nan=True), (i, j)
            assert (np.abs(got[r][fine] - want[fine]) <= bound[fine]).all(), (i, j)


HEADS = [(14, 2, 64), (28, 4, 128), (8, 8, 32), (24, 8, 96)]
# window, sinks, and positions of 1000: in the sinks' tile, where the window begins, in whole
# tiles, among the last ones
PLACES = [(300, 5, (1, 4, 705, 730, 800, 863, 960, 995)), (2 ** 31 - 1, 0, (0, 31, 500, 992, 998))]


# 21 and 161 K/V tiles, cut in chunks of 5: the last one holds one tile, and that one position
@pytest.mark.parametrize("heads,ctx,new", [((14, 2, 64), 641, 1), ((14, 2, 64), 5121, 1),
                                           ((28, 4, 128), 641, 2), ((28, 4, 128), 5121, 2),
                                           ((24, 8, 96), 641, 1), ((28, 4, 128), 641, 40)])
@pytest.mark.parametrize("value", ["k", "v"])
def test_last_position_of_many_chunks(heads, ctx, new, value):
    """Walks in chunks whose last one holds the newest position alone, which is NaN."""
    b = Batch(heads, [ctx], [new], 64, 2 ** 31 - 1, 0, seed=ctx)
    assert b.need()
    put(b, 0, ctx - 1, slice(None), slice(None), **{value: NAN})
    got = b.run()
    assert np.isnan(got[new - 1]).all()
    check(b, got)
