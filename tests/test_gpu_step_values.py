"""Infinities and NaN that a row of si_attention_rows sees: the outputs that the definition gives,
wherever the position lies in the walk and however the walk is cut."""
import numpy as np
import pytest

import si_amd
from tests import step_ref
from tests.gpu_helpers import torch_cuda
from tests.test_gpu_step import P, Batch, host, st

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


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("new", [1, 6, 40])
@pytest.mark.parametrize("window,sinks,places", PLACES)
def test_values_that_are_seen(heads, page, new, window, sinks, places):
    """Infinities of either sign, both, and NaN in V, one value each: that value alone is not
    finite, and has the sign that the definition gives."""
    b = Batch(heads, [1000, 90], [new, 1], page, window, sinks, seed=new)
    g, D = heads[1], heads[2]
    for n, pos in enumerate(places):
        put(b, 0, pos, n % g, (3 * n) % D, v=[INF, -INF, NAN, INF][n % 4])
        put(b, 0, pos, (n + 1) % g, D - 1, v=[INF, -INF][n % 2])
    put(b, 1, 50, 0, 1, v=-INF)
    check(b, b.run())


@pytest.mark.parametrize("heads", HEADS[:2])
@pytest.mark.parametrize("new", [1, 6, 40])
@pytest.mark.parametrize("window,sinks,places", PLACES)
def test_keys_that_are_seen(heads, new, window, sinks, places):
    """An infinite key: the heads that it meets with a negative q give it no weight, the others are
    NaN; so is a head that meets a NaN."""
    for n, pos in enumerate(places):
        b = Batch(heads, [1000, 90], [new, 1], 16, window, sinks, seed=n)
        put(b, 0, pos, 0, n, k=[INF, -INF][n % 2], v=[None, 2.0, INF][n % 3])
        put(b, 1, 60, 0, 5, k=NAN)
        check(b, b.run())


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


@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_values_far_below_the_largest(value):
    """A position whose weight is next to nothing in 32 bits gives its infinity all the same, in
    its own tile, wavefront and chunk."""
    heads = (12, 2, 128)
    for new, at in ((1, 3), (1, 700), (1, 1500), (12, 700)):
        b = Batch(heads, [3000], [new], 64, 2 ** 31 - 1, 0, seed=7)
        # the last 100 positions' scores lie 200 and more above the others'
        top = b.q.reshape(-1, 2, 6, 128).sum((0, 2))
        top /= np.linalg.norm(top, axis=-1, keepdims=True)
        b.q += 6 * top[None, :, None].repeat(6, 2).reshape(1, 12, 128)
        for pos in range(2900, 3000):
            put(b, 0, pos, slice(None), slice(None), k=(top * 500).astype(np.float16))
        put(b, 0, at, 1, 9, v=value)
        check(b, b.run())


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("new", [1, 6, 40])
def test_quantized_around_them(heads, new):
    """The Q8_0 of blocks without such values, of the rows that have them and of their neighbours, as
    si_quantize_q8_rows has it."""
    torch = torch_cuda()
    b = Batch(heads, [400, 90], [new, 1], 16, 300, 4, seed=new)
    put(b, 0, 398 - new // 2, 0, 3, v=INF)
    put(b, 0, 200, 1, heads[2] - 1, v=NAN)
    b.upload()
    n, qd = b.max_rows, heads[0] * heads[2]
    out = torch.full((n, qd), 7.0, device="cuda")
    bufs = [torch.full((n, qd), 7, dtype=torch.int8, device="cuda"),
            *(torch.full((n, qd // 32), 7, dtype=torch.int16, device="cuda") for _ in range(2))]
    b.call(out, bufs)
    fine = torch.isfinite(out).view(n, -1, 32).all(2)
    assert not fine.all() and fine.any(1).all()
    clean = torch.where(torch.isfinite(out), out, 0.0).contiguous()
    want = [torch.empty_like(x) for x in bufs]
    si_amd.call("si_quantize_q8_rows", P(clean), n, qd, *(P(x) for x in want), st())
    assert torch.equal(bufs[0].view(n, -1, 32)[fine], want[0].view(n, -1, 32)[fine])
    for x, y in zip(bufs[1:], want[1:]):
        assert torch.equal(x[fine], y[fine])
    check(b, host(out).reshape(n, *heads[::2]))


def test_values_between_replays():
    """One captured call, whose pools hold such values in some replays: each is the eager call's."""
    torch = torch_cuda()
    heads = (28, 4, 128)
    for new in ([1, 1], [6, 2], [50, 1]):
        b = Batch(heads, [1500, 300], new, 16, 1000, 4, seed=new[0])
        pools = []
        for value in (None, INF, NAN, None, -INF):
            if value is not None:
                put(b, 0, 1490, 1, 7, v=value)
                put(b, 1, 200, 2, 9, k=value)
            want = b.run()
            pools.append((b.dk.clone(), b.dv.clone(), want))
            put(b, 0, 1490, 1, 7, v=0.5)
            put(b, 1, 200, 2, 9, k=0.5)
        out, side, graph = torch.full_like(b.out, 7.0), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            b.call(out, ws=b.ws)
        for k in (0, 1, 0, 2, 3, 4, 1, 0):
            dk, dv, want = pools[k]
            b.dk.copy_(dk)
            b.dv.copy_(dv)
            out.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(host(out).reshape(want.shape), want, equal_nan=True), (new, k)
