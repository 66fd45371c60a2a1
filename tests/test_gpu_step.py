"""A ragged step's page lists, append and windowed attention against plain numpy, and a run of
them together."""
import ctypes

import numpy as np
import pytest

import si_amd
from tests import step_ref
from tests.gpu_helpers import dev, torch_cuda

pytestmark = pytest.mark.gpu

HEADS = [(14, 2, 64), (28, 4, 128), (8, 8, 32), (24, 8, 96), (16, 1, 128)]
P = si_amd.ptr


def st():
    return si_amd.stream_handle()


def shape_of(heads):
    return ctypes.byref(si_amd.make_shape(32, *heads))


def host(t):
    return t.cpu().numpy()


# ---------------------------------------------------------------------------
# page lists and slot maps
# ---------------------------------------------------------------------------
class Tables:
    """A step's device arrays and their call."""

    def __init__(self, nseq, page, npages, max_pages, max_rows, window, sinks, seed=0):
        rng = np.random.default_rng(seed)
        self.sizes = (nseq, page, npages, max_pages, max_rows, window, sinks)
        i32 = np.int32
        self.pages = dev(np.full((max(nseq, 1), max_pages), -7, i32))
        self.ring = dev(rng.permutation(npages).astype(i32))
        self.free = dev(np.array([rng.integers(npages), npages], i32))
        self.held = dev(np.zeros((max(nseq, 1), 2), i32))
        self.start, self.taken = (dev(np.full(nseq + 1, -9, i32)) for _ in range(2))
        self.ctx = dev(np.full(max(nseq, 1), -9, i32))
        self.seq, self.pos = (dev(np.full(max(max_rows, 1), -9, i32)) for _ in range(2))
        self.slot = dev(np.full(max(max_rows, 1), -9, np.int64))
        self.status = dev(np.full(4, -9, i32))

    def run(self, have, add, free_out=None, held_out=None):
        nseq, page, npages, max_pages, max_rows, window, sinks = self.sizes
        self.have, self.add = have, add
        si_amd.call("si_kv_step", nseq, P(have), P(add), max_rows, window, sinks, page, npages,
                    max_pages, P(self.pages), P(self.ring), P(self.free),
                    P(self.free if free_out is None else free_out), P(self.held),
                    P(self.held if held_out is None else held_out), P(self.start), P(self.ctx),
                    P(self.seq), P(self.pos), P(self.slot), P(self.taken), P(self.status), st())

    def ref(self, have, add):
        nseq, page, npages, max_pages, max_rows, window, sinks = self.sizes
        return step_ref.tables(have, add, host(self.held)[:nseq], host(self.pages)[:nseq],
                               host(self.ring), host(self.free), page, window, sinks, max_rows)

    def check(self, want, free=None, held=None):
        nseq, max_rows = self.sizes[0], self.sizes[4]
        got = dict(pages=self.pages[:nseq], ring=self.ring, free=free, held=held,
                   start=self.start, ctx=self.ctx[:nseq], seq=self.seq[:max_rows],
                   pos=self.pos[:max_rows], slot=self.slot[:max_rows], taken=self.taken,
                   status=self.status)
        got["free"] = self.free if free is None else free
        got["held"] = (self.held if held is None else held)[:nseq]
        for k, t in got.items():
            assert np.array_equal(host(t), want[k]), k


def lengths(rng, nseq, add_most, have_most):
    return (rng.integers(0, have_most + 1, nseq).astype(np.int32),
            rng.integers(0, add_most + 1, nseq).astype(np.int32))


@pytest.mark.parametrize("nseq,page,window,sinks,add_most", [
    (0, 16, 8, 4, 1), (1, 16, 100, 4, 5), (1, 1, 1, 0, 3), (2, 4, 2 ** 31 - 1, 0, 9),
    (63, 16, 20, 4, 1), (64, 16, 33, 17, 8), (65, 64, 64, 0, 3), (300, 1, 7, 3, 4),
    (1023, 4, 10, 4, 2), (1024, 16, 16, 16, 2), (1025, 16, 31, 33, 2), (2500, 32, 40, 4, 3),
    (5, 16, 50, 4, 3000), (40, 8, 100, 9, 400)])
@pytest.mark.parametrize("apart", [False, True])
def test_tables_over_steps(nseq, page, window, sinks, add_most, apart):
    """Steps in a row: rows taken in, drafts refused again, sequences that end and begin, every
    number of every step; no page in two places."""
    rng = np.random.default_rng(nseq + page)
    steps, most = 6, add_most * 7 + 3 * page
    max_pages = -(-most // page) + 1
    npages = max(1, nseq * max_pages + 5)
    max_rows = nseq * add_most + 3
    t = Tables(nseq, page, npages, max_pages, max_rows, window, sinks)
    have = np.zeros(nseq, np.int32)
    for step in range(steps):
        add = rng.integers(0, add_most + 1, nseq).astype(np.int32)
        add[rng.random(nseq) < 0.1] = -3
        want = t.ref(have, add)
        free, held = (x.clone() for x in (t.free, t.held)) if apart else (None, None)
        t.run(dev(have), dev(add), free, held)
        t.check(want, free, held)
        if apart:
            t.free, t.held = free, held
        assert want["status"][0] == 0
        h, f, r, pg = host(t.held), host(t.free), host(t.ring), host(t.pages)
        kept = -(-sinks // page)
        own = [pg[i, j] for i in range(nseq) for j in range(h[i, 0])
               if j < kept or j >= kept + h[i, 1]]
        own += [r[(f[0] + k) % npages] for k in range(f[1])]
        assert sorted(own) == list(range(npages))
        # some drafts are refused, some sequences end (and begin anew in the step after)
        ended = have < 0
        have = np.maximum(have, 0) + np.maximum(add, 0) * (have >= 0)
        have = (have - np.minimum(rng.integers(0, 3, nseq), np.maximum(add, 0) * ~ended))
        have = have.astype(np.int32)
        have[rng.random(nseq) < 0.1] = -1
        have[ended] = 0


def filled(nseq=4, page=4, npages=20, max_pages=4, max_rows=8, window=100, sinks=0):
    t = Tables(nseq, page, npages, max_pages, max_rows, window, sinks)
    have, add = np.zeros(nseq, np.int32), np.full(nseq, 2, np.int32)
    t.run(dev(have), dev(add))
    return t, have + 2


@pytest.mark.parametrize("change,add,code", [
    ({}, [2, 2, 2, 3], 1), ({}, [8, 1, 1, 1], 1), (dict(npages=5), [3, 3, 0, 0], 2),
    (dict(npages=4), [0, 0, 0, 3], 2), ({}, [15, 0, 0, 0], 4), ({}, [2 ** 31 - 1, 0, 0, 0], 4),
    (dict(npages=4), [15, 3, 3, 3], 7)])
def test_tables_refused(change, add, code):
    """A step that does not fit has no rows, takes nothing and gives nothing back."""
    t, have = filled(**change)
    before = [host(x).copy() for x in (t.pages, t.ring, t.free, t.held)]
    want = t.ref(have, np.array(add, np.int32))
    t.run(dev(have), dev(np.array(add, np.int32)))
    t.check(want)
    assert host(t.status)[0] == code and (host(t.slot) == -1).all()
    for a, b in zip(before, (t.pages, t.ring, t.free, t.held)):
        assert np.array_equal(a, host(b))


def test_tables_positions_without_pages():
    t, have = filled()
    have[2] = 5  # of one page of 4
    want = t.ref(have, np.array([1, 1, 1, 1], np.int32))
    t.run(dev(have), dev(np.array([1, 1, 1, 1], np.int32)))
    t.check(want)
    assert host(t.status)[0] == 4


def test_tables_state_out_of_range():
    """Numbers that no step left: nothing outside the arrays is touched, ids stay in the pool."""
    t, have = filled()
    t.held.copy_(dev(np.array([[99, 99], [-5, 3], [1, -2], [1, 50]], np.int32)))
    t.free.copy_(dev(np.array([1000, 1 << 30], np.int32)))
    t.ring.fill_(1 << 20)
    t.run(dev(have), dev(np.ones(4, np.int32)))
    slot = host(t.slot)
    assert ((slot >= -1) & (slot < 20 * 4)).all()
    f = host(t.free)
    assert 0 <= f[0] < 20 and 0 <= f[1] <= 20


def test_tables_more_pages_than_there_are():
    """A ring and lists that together hold more than the pool: refused, nothing changes."""
    t, have = filled()
    t.free.copy_(dev(np.array([3, 20], np.int32)))  # all free, and four taken
    before = [host(x).copy() for x in (t.pages, t.ring, t.free, t.held)]
    have[1] = -1
    t.run(dev(have), dev(np.zeros(4, np.int32)))
    assert host(t.status).tolist() == [4, 0, 0, 0]
    for a, b in zip(before, (t.pages, t.ring, t.free, t.held)):
        assert np.array_equal(a, host(b))


def test_tables_long_prompt():
    """One sequence of many pages next to idle ones."""
    t = Tables(70, 1, 300000, 250000, 260000, 1000, 4)
    have, add = np.zeros(70, np.int32), np.zeros(70, np.int32)
    add[33], add[34] = 200001, 7
    want = t.ref(have, add)
    t.run(dev(have), dev(add))
    t.check(want)
    have, add = add.copy(), np.ones(70, np.int32)
    want = t.ref(have, add)
    t.run(dev(have), dev(add))
    t.check(want)
    assert want["status"][3] == 200001 - 1000 + 1 - 4


# ---------------------------------------------------------------------------
# the append
# ---------------------------------------------------------------------------
def rope_table(n, D):
    c, s = (np.empty((n, D // 2), np.float32) for _ in range(2))
    si_amd.call("si_rope_table", n, D, 1e6, P(c), P(s))
    return dev(c), dev(s)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("rows,extra", [(1, 0), (5, 3), (67, 1), (300, 0)])
def test_append_bits(heads, rows, extra):
    """The bits of si_rope_kv_append, wherever the slots lie; rows without a position or a place
    are left as they were, in q and in the pools."""
    torch = torch_cuda()
    q, kv, D = heads
    rng = np.random.default_rng(rows)
    ld, n, npos = (q + 2 * kv) * D + extra, 2 * rows + 9, rows + 40
    qkv = dev(rng.standard_normal((rows, ld)).astype(np.float32))
    qkv[rows // 2, :] *= 1e5  # past fp16's largest
    c, s = rope_table(npos, D)
    first = int(rng.integers(0, 40))
    q_ref = torch.zeros(rows, q * D, device="cuda")
    kc, vc = (torch.zeros(npos, kv * D, dtype=torch.float16, device="cuda") for _ in range(2))
    si_amd.call("si_rope_kv_append", ctypes.byref(si_amd.make_shape(32, *heads)), P(qkv), ld,
                rows, first, 1, npos, None, P(c), P(s), P(q_ref), P(kc), P(vc), 0, st())
    slot = rng.permutation(n)[:rows].astype(np.int64)
    pos = (first + np.arange(rows)).astype(np.int32)
    dead = rng.random(rows) < 0.2
    bad_slot, bad_pos = slot.copy(), pos.copy()
    for i in np.nonzero(dead)[0]:
        if i % 2:
            bad_slot[i] = [-1, n, 2 ** 40][i % 3]
        else:
            bad_pos[i] = [-1, npos, 2 ** 31 - 1][i % 3]
    q_out = torch.full((rows, q * D), 7.0, device="cuda")
    k, v = (torch.full((n, kv * D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    si_amd.call("si_rope_kv_append_rows", shape_of(heads), P(qkv), ld, rows, npos,
                P(dev(bad_pos)), P(dev(bad_slot)), P(c), P(s), P(q_out), P(k), P(v), n, st())
    for got, ref in ((k, kc), (v, vc)):
        want = np.full((n, kv * D), 7.0, np.float16)
        want[slot[~dead]] = host(ref)[first:first + rows][~dead]
        assert np.array_equal(host(got).view(np.uint16), want.view(np.uint16))
    want = np.full((rows, q * D), 7.0, np.float32)
    want[~dead] = host(q_ref)[~dead]
    assert np.array_equal(host(q_out).view(np.uint32), want.view(np.uint32))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
class Batch:
    """Rows over pages: sequences of contexts ctx with new rows each, pages in random order, the
    entries behind the window stale."""

    def __init__(self, heads, ctx, new, page, window, sinks, seed=0, room=0, max_ctx=None,
                 max_new=None, garbage=np.nan):
        rng = np.random.default_rng(seed)
        q, kv, D = heads
        self.heads, self.page, self.window, self.sinks = heads, page, window, sinks
        self.ctx, self.new = np.array(ctx), np.array(new)
        n = len(ctx)
        self.rows = int(self.new.sum())
        self.max_rows = self.rows + room
        self.max_ctx = max_ctx or max(1, int(self.ctx.max()))
        self.max_new = max_new or max(1, int(self.new.max()))
        self.start = np.concatenate([[0], np.cumsum(self.new)])
        self.max_pages = -(-max(self.max_ctx, int(self.ctx.max())) // page)
        used = [-(-int(c) // page) for c in self.ctx]
        self.npages = sum(used) + 1
        ids = rng.permutation(self.npages)
        self.pages = rng.integers(0, self.npages, (n, self.max_pages))
        self.q = rng.standard_normal((self.max_rows, q, D)).astype(np.float32)
        # (what no sequence holds is not a number)
        self.kpool, self.vpool = (np.full((self.npages, page, kv, D), garbage, np.float16)
                                  for _ in range(2))
        self.k, self.v = [], []
        at = 0
        for i, c in enumerate(self.ctx):
            k, v = (rng.standard_normal((int(c), kv, D)).astype(np.float16) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            for j in range(used[i]):
                part = slice(j * page, min((j + 1) * page, int(c)))
                self.pages[i, j] = ids[at]
                at += 1
                self.kpool[self.pages[i, j], :part.stop - part.start] = k[part]
                self.vpool[self.pages[i, j], :part.stop - part.start] = v[part]
        # no row of this step sees the pages behind the first one's window
        for i in range(n):
            first = min(int(self.ctx[i]), self.max_ctx) - self.new[i] - window + 1
            for j in range(-(-sinks // page), max(0, int(first)) // page):
                self.pages[i, j] = rng.integers(-5, self.npages + 5)

    def upload(self):
        self.dq = dev(self.q.reshape(self.max_rows, -1))
        self.dk, self.dv = dev(self.kpool), dev(self.vpool)
        self.dp = dev(self.pages.astype(np.int32))
        self.ds, self.dc = dev(self.start.astype(np.int32)), dev(self.ctx.astype(np.int32))
        return self

    def sizes(self):
        return (len(self.ctx), self.max_rows, self.max_new, self.max_ctx, self.window, self.sinks)

    def need(self):
        return si_amd.lib().si_attention_rows_workspace(shape_of(self.heads), *self.sizes())

    def call(self, out, quant=(None, None, None), ws=None, stream=None):
        torch = torch_cuda()
        need = self.need()
        if ws is None:
            self.ws = torch.full((max(need, 256),), 255, dtype=torch.uint8, device="cuda")
        si_amd.call("si_attention_rows", shape_of(self.heads), P(self.dq), *self.sizes(),
                    P(self.ds), P(self.dc), P(self.dk), P(self.dv), self.npages, self.page,
                    P(self.dp), self.max_pages, P(out), *(P(x) for x in quant),
                    P(self.ws if ws is None else ws), need, stream or st())

    def run(self):
        torch = torch_cuda()
        self.upload()
        self.out = torch.full((self.max_rows, self.heads[0] * self.heads[2]), 7.0, device="cuda")
        self.call(self.out)
        torch.cuda.synchronize()
        return host(self.out).reshape(self.max_rows, *self.heads[::2])

    def check(self, got, every=1):
        """Every row (or some of the many) against 64 bits; the others as they were."""
        off = size = may = 0.0
        for i in range(len(self.ctx)):
            n = min(int(self.new[i]), self.max_new)
            c = min(int(self.ctx[i]), self.max_ctx)
            s = int(self.start[i])
            js = range(n) if n <= 8 else sorted({0, 1, n // 2, n - 2, n - 1, *range(0, n, every)})
            for j in js:
                want, bound = step_ref.attend(self.q[s + j], self.k[i], self.v[i],
                                              c - int(self.new[i]) + j, self.window, self.sinks,
                                              self.heads[0] // self.heads[1])
                err = np.abs(got[s + j] - want)
                assert (err <= bound).all(), (i, j, err.max(), bound[err > bound])
                off, size = off + (err ** 2).sum(), size + (want ** 2).sum()
                # roundings of either sign add up as a walk does: n positions' sums by
                # 2^-24 sqrt(n) of the result, whose size is a walk's too; scores of about 3,
                # from D products, by 2^-24 of it sqrt(D) times, 16 for the rest
                seen = step_ref.visible(c - int(self.new[i]) + j, self.window, self.sinks).size
                part = 2.0 ** -24 * (seen ** 0.5 + 3 * self.heads[2] ** 0.5 + 16)
                may += part ** 2 * (want ** 2).sum()
            assert (got[s + n:int(self.start[i + 1])] == 7.0).all()
        assert (got[self.rows:] == 7.0).all()
        assert off <= may, ((off / size) ** 0.5, (may / size) ** 0.5)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page,window,sinks,ctx,new", [
    (16, 2 ** 31 - 1, 0, [1], [1]),
    (16, 20, 4, [1, 2, 33, 31, 100], [1, 1, 1, 1, 1]),
    (1, 5, 0, [64, 7, 3], [3, 7, 0]),
    (4, 33, 1, [200, 5, 64, 65], [2, 5, 1, 9]),
    (32, 64, 40, [300, 64, 129], [1, 1, 1]),
    (64, 1, 0, [150, 3], [4, 1]),
    (64, 1, 3, [150, 3], [4, 1]),
    (128, 100, 4, [777, 130, 0, 258], [5, 8, 0, 1]),
    (16, 90, 70, [333, 40], [200, 40]),
    (64, 2 ** 31 - 1, 0, [500], [130]),
    (256, 300, 4, [1500, 1499], [1, 2])])
def test_attention(heads, page, window, sinks, ctx, new):
    b = Batch(heads, ctx, new, page, window, sinks, seed=sum(ctx), room=3)
    b.check(b.run(), every=13)


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (12, 2, 128), (32, 2, 64)])
@pytest.mark.parametrize("n", [1, 2, 7, 40])
def test_attention_long_rows(heads, n):
    """Few rows over long ranges, whose ends differ."""
    rng = np.random.default_rng(n)
    ctx = rng.integers(1, 6000, n)
    ctx[0] = 6001
    b = Batch(heads, ctx, np.minimum(ctx, rng.integers(0, 4, n)), 64, 2500, 4, seed=n)
    b.check(b.run())


@pytest.mark.parametrize("heads", HEADS)
def test_attention_prompts(heads):
    """Pieces of prompts among single tokens, from the start of their sequences and after it."""
    b = Batch(heads, [700, 1, 900, 450, 33, 2000], [700, 1, 1, 333, 20, 64], 64, 256, 4, seed=5,
              room=7)
    b.check(b.run(), every=37)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 65504.0])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [1, 6, 90])
def test_attention_hidden_values(bad, page, new):
    """What a row does not see has no influence on it: the rows of later tokens, and positions
    behind the window that a neighbour still sees."""
    heads, window, sinks, L = (14, 2, 64), 70, 4, 400
    b = Batch(heads, [L, 50], [new, 1], page, window, sinks, seed=new, garbage=bad)
    clean = b.run()
    b.check(clean, every=7)
    # the rows at first and last: what only one of them sees is bad
    for at, bent in ((L - 1, range(new - 1, new)), (L - new - window + 1, range(1))):
        k, v = b.kpool.copy(), b.vpool.copy()
        slot = b.pages[0, at // page], at % page
        b.kpool[slot], b.vpool[slot] = bad, bad
        got = b.run()
        keep = np.ones(b.max_rows, bool)
        keep[list(bent)] = False
        assert np.array_equal(got[keep], clean[keep]), at
        if not np.isfinite(bad):
            assert not np.isfinite(got[~keep]).any()
        b.kpool, b.vpool = k, v


def test_attention_rows_before_the_start():
    """More rows than positions: those before position 0 see nothing and are zeros."""
    b = Batch((14, 2, 64), [3, 40], [5, 2], 16, 100, 4, max_new=5)
    got = b.run()
    assert (got[:2] == 0).all()
    b.check(got)


def test_attention_starts_past_the_rows():
    """A last sequence that reaches past max_rows: the rows that are there, at their positions."""
    for new in ([3, 40], [3, 5]):
        b = Batch((14, 2, 64), [60, 90], new, 16, 50, 4, seed=3)
        b.upload()
        b.max_rows = b.rows - 3
        b.out = dev(np.full((b.max_rows + 4, 14 * 64), 7.0, np.float32))
        b.call(b.out)
        got = host(b.out).reshape(-1, 14, 64)
        assert (got[b.max_rows:] == 7.0).all()
        b.rows = b.max_rows
        b.new[1] -= 3
        b.ctx[1] -= 3
        b.start[2] -= 3
        b.check(got[:b.max_rows], every=3)


def test_attention_starts_that_are_none():
    """Starts in no order, below 0 and past the rows: every row that is written is one of some
    sequence (values are the caller's affair), those behind max_rows are left as they are."""
    rng = np.random.default_rng(6)
    for max_new in (2, 64):
        b = Batch((14, 2, 64), [60, 90, 40, 30], [20, 20, 1, 3], 16, 50, 4, max_new=max_new)
        b.upload()
        for _ in range(4):
            b.ds = dev(rng.integers(-50, 100, 5).astype(np.int32))
            b.dc = dev(rng.integers(-20, 200, 4).astype(np.int32))
            out = dev(np.full((b.max_rows + 4, 14 * 64), 7.0, np.float32))
            b.call(out)
            assert (host(out)[b.max_rows:] == 7.0).all()


def test_attention_limits():
    """Contexts past max_ctx are max_ctx; rows past max_new are left as they are."""
    b = Batch((14, 2, 64), [100, 90, 64], [9, 2, 3], 16, 50, 4, max_ctx=64, max_new=4)
    b.check(b.run())


def test_attention_quantized():
    """The Q8_0 of the outputs, as si_quantize_q8_rows has it."""
    torch = torch_cuda()
    for heads, new in (((28, 4, 128), [1, 5, 0, 1]), ((24, 8, 96), [200, 1, 1, 1])):
        b = Batch(heads, [900, 70, 64, 400], new, 32, 128, 4, room=2).upload()
        qd = heads[0] * heads[2]
        n = b.max_rows
        bufs = []
        for _ in range(2):
            bufs.append([torch.full((n, qd), 7.0, device="cuda"),
                         torch.full((n, qd), 7, dtype=torch.int8, device="cuda"),
                         torch.full((n, qd // 32), 7, dtype=torch.int16, device="cuda"),
                         torch.full((n, qd // 32), 7, dtype=torch.int16, device="cuda")])
        b.call(bufs[0][0], bufs[0][1:])
        b.call(bufs[1][0], (bufs[1][1], bufs[1][2], None))
        qs, d, s = (torch.empty_like(x) for x in bufs[0][1:])
        si_amd.call("si_quantize_q8_rows", P(bufs[0][0]), n, qd, P(qs), P(d), P(s), st())
        for got, want in zip(bufs[0][1:], (qs, d, s)):
            assert torch.equal(got[:b.rows], want[:b.rows])
            assert (got[b.rows:] == 7).all()
        assert torch.equal(bufs[0][1], bufs[1][1]) and torch.equal(bufs[0][2], bufs[1][2])
        assert (bufs[1][3] == 7).all()


def test_attention_large_pool():
    """Pages past 2^32 bytes of their pool."""
    torch = torch_cuda()
    heads, page = (8, 8, 32), 1 << 20
    b = Batch(heads, [40, 70], [1, 3], 1, 30, 4)
    rows = 10 * page  # 512 bytes each
    k, v = (torch.zeros(rows, 256, dtype=torch.float16, device="cuda") for _ in range(2))
    b.upload()
    pages = dev(np.array([[9], [8]], np.int32))
    for i, c in enumerate(b.ctx):
        at = int(pages[i, 0]) * page
        k[at:at + c] = dev(b.k[i]).view(-1, 256)
        v[at:at + c] = dev(b.v[i]).view(-1, 256)
    b.dk, b.dv, b.dp, b.npages, b.page, b.max_pages = k, v, pages, 10, page, 1
    out = torch.full((b.max_rows, 256), 7.0, device="cuda")
    b.call(out)
    b.check(host(out).reshape(b.max_rows, 8, 32))


def test_attention_large_queries():
    """Queries of any size, and scores far apart."""
    for scale in (1e-30, 1e-4, 30.0, 3e4):
        b = Batch((14, 2, 64), [300, 40], [3, 1], 16, 200, 4)
        b.q *= scale
        got = b.run()
        assert np.isfinite(got).all()
        if scale < 1000:
            b.check(got)


def test_attention_sink_far_above():
    """A first position whose score lies far above the others' and whose values are zero (an
    attention sink) leaves the others' weights their bits."""
    for nats in (5.0, 12.0, 20.0):
        b = Batch((12, 2, 128), [500, 700], [1, 40], 16, 200, 1, seed=9)
        direction = b.q.reshape(b.max_rows, 2, 6, 128).sum((0, 2))
        for i in range(2):
            b.k[i][0] = (direction / np.linalg.norm(direction, axis=-1, keepdims=True)
                         * 8).astype(np.float16)
            b.v[i][0] = 0
            slot = b.pages[i, 0], 0
            b.kpool[slot], b.vpool[slot] = b.k[i][0], 0
            # every query meets it with the same score
            k0 = b.k[i][0].astype(np.float64)
            for r in range(b.start[i], b.start[i + 1]):
                for h in range(12):
                    x, kk = b.q[r, h].astype(np.float64), k0[h // 6]
                    have = x @ kk / np.sqrt(128)
                    b.q[r, h] = x + kk * (nats + 4 - have) * np.sqrt(128) / (kk @ kk)
        got = b.run()
        for i in range(2):
            for j in range(b.new[i]):
                r = b.start[i] + j
                want, _ = step_ref.attend(b.q[r], b.k[i], b.v[i], b.ctx[i] - b.new[i] + j, 200, 1,
                                          6)
                # scores of S = 30 and less from D products, whose 2^-24 are of either sign
                # (2 sqrt(D) 2^-24 S, 4e-5), and 2^-47 of the sink's weight at each of 200
                # others, which are e^-(nats + 4) of it
                tol = 4e-5 + 200 ** 0.5 * 2.0 ** -47 * np.exp(nats + 4)
                rel = np.linalg.norm(got[r] - want) / np.linalg.norm(want)
                assert rel <= tol, (nats, r, rel, tol)


def test_attention_repeats():
    """The same bits from call to call, also over a workspace that other calls used."""
    torch = torch_cuda()
    b = Batch((28, 4, 128), [4000, 3000, 90, 5000], [1, 4, 30, 1], 64, 2048, 4)
    first = b.run()
    for fill in (0, 255):
        b.ws.fill_(fill)
        out = torch.full_like(b.out, 7.0)
        b.call(out, ws=b.ws)
        assert np.array_equal(host(out).reshape(first.shape), first)


def test_attention_on_another_stream():
    torch = torch_cuda()
    b = Batch((14, 2, 64), [3000, 30], [1, 5], 16, 1024, 4)
    want = b.run()
    side = torch.cuda.Stream()
    out = torch.full_like(b.out, 7.0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.call(out, ws=b.ws)
    side.synchronize()
    assert np.array_equal(host(out).reshape(want.shape), want)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
class Server:
    """Tables, append and attention, over caches that the test also keeps in numpy."""

    def __init__(self, heads, nseq, page, npages, max_pages, max_rows, max_new, window, sinks):
        torch = torch_cuda()
        q, kv, D = heads
        self.heads, self.window, self.sinks, self.max_new = heads, window, sinks, max_new
        self.max_rows, self.max_ctx = max_rows, max_pages * page
        self.t = Tables(nseq, page, npages, max_pages, max_rows, window, sinks, seed=3)
        self.have, self.add = (torch.zeros(nseq, dtype=torch.int32, device="cuda")
                               for _ in range(2))
        self.qkv = torch.zeros(max_rows, (q + 2 * kv) * D, device="cuda")
        self.cos, self.sin = rope_table(self.max_ctx, D)
        self.q = torch.zeros(max_rows, q * D, device="cuda")
        self.k, self.v = (torch.full((npages * page, kv * D), float("nan"), dtype=torch.float16,
                                     device="cuda") for _ in range(2))
        self.out = torch.full((max_rows, q * D), 7.0, device="cuda")
        sizes = (nseq, max_rows, max_new, self.max_ctx, window, sinks)
        need = si_amd.lib().si_attention_rows_workspace(shape_of(heads), *sizes)
        self.ws = torch.zeros(max(need, 256), dtype=torch.uint8, device="cuda")
        self.sizes, self.need, self.npages, self.page = sizes, need, npages, page
        self.max_pages = max_pages

    def step(self):
        t = self.t
        t.run(self.have, self.add)
        si_amd.call("si_rope_kv_append_rows", shape_of(self.heads), P(self.qkv),
                    self.qkv.shape[1], self.max_rows, self.max_ctx, P(t.pos), P(t.slot),
                    P(self.cos), P(self.sin), P(self.q), P(self.k), P(self.v), self.k.shape[0],
                    st())
        si_amd.call("si_attention_rows", shape_of(self.heads), P(self.q), *self.sizes, P(t.start),
                    P(t.ctx), P(self.k), P(self.v), self.npages, self.page, P(t.pages),
                    self.max_pages, P(self.out), None, None, None, P(self.ws), self.need, st())


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("heads,page", [((14, 2, 64), 16), ((12, 2, 128), 64), ((24, 8, 96), 8)])
def test_steps_together(heads, page, captured):
    """Prompts, single tokens, drafts that are refused, sequences that end and others in their
    place, from a pool that holds windows and not whole sequences: every step's outputs, eager
    or from one captured graph."""
    torch = torch_cuda()
    q, kv, D = heads
    nseq, window, sinks, max_new = 5, 3 * page + 5, 3, 4 * page + 1
    s = Server(heads, nseq, page, 40, 16, 6 * page, max_new, window, sinks)
    rng = np.random.default_rng(page)
    cos, sin = host(s.cos).astype(np.float64), host(s.sin).astype(np.float64)
    if captured:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            s.add.zero_()
            s.step()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                s.step()
        torch.cuda.synchronize()
    have = np.zeros(nseq, np.int32)
    keys = [np.zeros((0, kv, D)) for _ in range(nseq)]
    values = [np.zeros((0, kv, D)) for _ in range(nseq)]
    for step in range(9):
        add = rng.integers(0, 6, nseq).astype(np.int32)
        if step % 3 == 0:
            add[step // 3] = 4 * page + 1 if have[step // 3] == 0 else 2 * page
        if step == 5:
            have[1] = -1
        s.have.copy_(dev(have))
        s.add.copy_(dev(add))
        qkv = rng.standard_normal((s.max_rows, (q + 2 * kv) * D)).astype(np.float32)
        s.qkv.copy_(dev(qkv))
        s.out.fill_(7.0)
        if captured:
            torch.cuda.synchronize()
            graph.replay()
        else:
            s.step()
        torch.cuda.synchronize()
        assert host(s.t.status)[0] == 0
        got, r = host(s.out).reshape(-1, q, D), 0
        for i in range(nseq):
            if have[i] < 0:
                keys[i], values[i] = keys[i][:0], values[i][:0]
                have[i] = 0
                continue
            x = qkv[r:r + add[i]].reshape(-1, q + 2 * kv, D).astype(np.float64)
            p = have[i] + np.arange(add[i])
            c, sn = cos[p][:, None], sin[p][:, None]
            a, b = x[..., :D // 2], x[..., D // 2:]
            y = np.concatenate([a * c - b * sn, b * c + a * sn], -1)
            keys[i] = np.concatenate([keys[i][:have[i]], y[:, q:q + kv]])
            values[i] = np.concatenate([values[i][:have[i]], x[:, q + kv:]])
            for j in range(add[i]):
                k16, v16 = keys[i].astype(np.float16), values[i].astype(np.float16)
                want, bound = step_ref.attend(y[j, :q], k16, v16, int(p[j]), window, sinks,
                                              q // kv)
                # an fp16 key from a 32-bit product may be a rounding (2^-10 of it between
                # neighbours) off this one's, for few of them: scores by 2^-10 of theirs
                err = np.linalg.norm(got[r + j] - want) / np.linalg.norm(want)
                assert err < 2.0 ** -10, (step, i, j, err)
            r += add[i]
            # up to two of the step's rows are refused again
            have[i] += add[i] - min(int(rng.integers(0, 3)), add[i])
        assert (got[r:] == 7.0).all()
