"""A ragged step at its limits: as many sequences as there may be, states that hold more pages than
the pool, small pages, two calls at once and two captured graphs over one workspace."""
import numpy as np
import pytest

import si_amd
from tests.gpu_helpers import dev, torch_cuda
from tests.test_gpu_step import Batch, Tables, filled, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("add_most,max_rows", [(1, 70000), (3, 120000), (0, 5)])
def test_tables_most_sequences(add_most, max_rows):
    """65535 sequences, two steps."""
    nseq = 65535
    rng = np.random.default_rng(add_most)
    t = Tables(nseq, 2, 200000, 3, max_rows, 1, 0)
    have = np.zeros(nseq, np.int32)
    for _ in range(2):
        add = rng.integers(0, add_most + 1, nseq).astype(np.int32)
        want = t.ref(have, add)
        t.run(dev(have), dev(add))
        t.check(want)
        have = (np.maximum(have, 0) + add).astype(np.int32)
        have[rng.random(nseq) < 0.1] = -1


def test_tables_too_many_pages_back():
    """Ids that would be given back over others that the same step takes: refused."""
    t, have = filled()
    t.free.copy_(dev(np.array([3, 20], np.int32)))  # all free, and four taken
    before = [host(x).copy() for x in (t.pages, t.ring, t.free, t.held)]
    have[1] = -1
    t.run(dev(have), dev(np.array([3, 0, 0, 0], np.int32)))
    assert host(t.status).tolist() == [4, 3, 1, 0]
    assert (host(t.slot) == -1).all()
    for a, b in zip(before, (t.pages, t.ring, t.free, t.held)):
        assert np.array_equal(a, host(b))


@pytest.mark.parametrize("new", [1, 30])
def test_attention_most_sequences(new):
    """65535 sequences of which few have rows."""
    ctx, rows = np.zeros(65535, np.int64), np.zeros(65535, np.int64)
    for i, (c, n) in {0: (90, 1), 7: (200, new), 40000: (33, 2), 65534: (150, new)}.items():
        ctx[i], rows[i] = c, n
    b = Batch((14, 2, 64), ctx, rows, 64, 100, 4, room=3)
    b.check(b.run())


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (24, 8, 96)])
@pytest.mark.parametrize("page", [2, 8])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 2, 90]])
def test_attention_small_pages(heads, page, new):
    b = Batch(heads, [65, 333, 700], new, page, 250, 5)
    b.check(b.run(), every=7)


def test_attention_two_at_once():
    """Calls on two streams, a workspace each."""
    torch = torch_cuda()
    b = [Batch((28, 4, 128), [4000, 3000, 90], [1, n, 3], 64, 2048, 4, seed=n) for n in (1, 60)]
    want = [x.run() for x in b]
    assert b[0].need() and b[1].need()
    streams = [torch.cuda.Stream() for _ in b]
    outs = [[torch.full_like(x.out, 7.0) for _ in range(5)] for x in b]
    torch.cuda.synchronize()
    for k in range(5):
        for x, s, o in zip(b, streams, outs):
            x.call(o[k], ws=x.ws, stream=si_amd.stream_handle(s))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for x in o:
            assert np.array_equal(host(x).reshape(w.shape), w)


def test_attention_graphs_share_a_workspace():
    """Two captured calls of other sizes over the same workspace, replayed in turn."""
    torch = torch_cuda()
    b = [Batch((28, 4, 128), [4000, 3000, 90], [1, n, 3], 64, 2048, 4, seed=n) for n in (1, 60)]
    want = [x.run() for x in b]
    ws = torch.full((max(x.need() for x in b),), 255, dtype=torch.uint8, device="cuda")
    graphs, side = [], torch.cuda.Stream()
    for x in b:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            x.call(x.out, ws=ws)
        graphs.append(g)
    for k in range(6):
        i = (k + k // 3) % 2
        b[i].out.fill_(7.0)
        torch.cuda.synchronize()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(b[i].out).reshape(want[i].shape), want[i]), k


@pytest.mark.parametrize("nseq,max_rows", [(1500, 4000), (20, 1800), (20, 60)])
def test_tables_replayed(nseq, max_rows):
    """One captured step over many: the state is taken on in place, whichever form runs."""
    torch = torch_cuda()
    rng = np.random.default_rng(nseq)
    page, window, sinks = 4, 9, 3
    t = Tables(nseq, page, nseq * 9, 12, max_rows, window, sinks)
    have, add = (torch.zeros(nseq, dtype=torch.int32, device="cuda") for _ in range(2))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        t.run(have, add)
    h = np.zeros(nseq, np.int32)
    for _ in range(6):
        a = rng.integers(0, 4, nseq).astype(np.int32)
        want = t.ref(h, a)
        assert want["status"][0] == 0
        have.copy_(dev(h))
        add.copy_(dev(a))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        t.check(want)
        h = (np.maximum(h, 0) + np.where(h < 0, 0, a)).astype(np.int32)
        h[rng.random(nseq) < 0.1] = -1


@pytest.mark.parametrize("ctx", [0, -1, -40, -2 ** 31 + 1, -2 ** 31])
@pytest.mark.parametrize("new,max_new", [([3, 1], 3), ([7, 1], 7), ([60, 1], 60)])
@pytest.mark.parametrize("last", [0, 2 ** 31 - 1])
def test_attention_contexts_below_zero(ctx, new, max_new, last):
    """Contexts that a sequence cannot have are 0: its rows lie before position 0 and are zeros,
    also where the starts are as far apart as they can be; its neighbour's are as ever."""
    b = Batch((14, 2, 64), [90, 90], new[::-1], 16, 50, 4, max_new=max_new)
    want = b.run()
    b.dc = dev(np.array([90, ctx], np.int32))
    if last:
        b.ds = dev(np.array([0, 1, last], np.int32))
    out = dev(np.full((b.max_rows + 2, 14 * 64), 7.0, np.float32))
    b.call(out)
    got = host(out).reshape(-1, 14, 64)
    assert np.array_equal(got[:1], want[:1])
    assert (got[1:b.max_rows] == 0).all() and (got[b.max_rows:] == 7.0).all()
