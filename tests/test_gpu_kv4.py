"""The K/V cache held in 4 bits on the GPU, against a plain 64-bit statement of it
(tests/kv4_ref.py).

Rows: q and the held K and V values are the reference's bits (RoPE and the block's
rule are exact operations on fp32 values); nothing else of a page changes.

Attention: q is taken as an fp16 pair, short of it by at most 2^-22 of its value,
the softmax's weights too; sums are fp32.  A score of magnitude S is then off by
about S (2^-22 + a few 2^-24), and a weight by that and the exponential's ulp: with
scores up to 30 that is 30 * 4 * 2^-24 = 7e-6 of a single weight, and the output, a
weighted mean, is off by at most that times the values' size (its rms in practice is
far below).  The bound below, 2e-5 of the row's largest value, is what a
fp32 result is held to."""
import ctypes

import numpy as np
import pytest

import si_amd
from tests import kv4_ref as ref
from tests.gpu_helpers import dev, empty, host, zeros

pytestmark = pytest.mark.gpu
SHAPES = {"g7_d64": (14, 2, 64), "g7_d128": (28, 4, 128), "g6_d128": (12, 2, 128),
          "g16_d64": (32, 2, 64), "g3_d96": (24, 8, 96), "g1_d32": (8, 8, 32),
          "g16_d128": (16, 1, 128), "g9_d32": (9, 1, 32), "g8_d96": (16, 2, 96)}
NAMES = list(SHAPES)


def _torch():
    import torch
    return torch


class Cache:
    """Random page lists over a pool of random bytes (finite scales), with spare pages."""

    def __init__(self, rng, name, nseq, longest, ps, fill=True):
        self.q, self.kv, self.D = SHAPES[name]
        self.ps, self.max_pages = ps, -(-longest // ps)
        self.npages = nseq * self.max_pages + 3
        self.pages = rng.permutation(self.npages)[:nseq * self.max_pages].reshape(
            nseq, -1).astype(np.int32)
        self.shape = si_amd.make_shape(32, self.q, self.kv, self.D)
        hb = ps * self.D * 9 // 16
        pools = rng.integers(0, 256, (2, self.npages, self.kv, hb), dtype=np.uint8)
        if fill:  # held rows; else bytes whose scales may be anything, NaN among them
            for i in (0, 1):
                x = rng.standard_normal((self.npages * ps, self.kv, self.D)).astype(np.float32)
                pools[i] = ref.pack(x * np.exp(rng.normal(0, 0.5, self.D)).astype(np.float32),
                                    self.kv, self.D, ps, i == 0)
        self.k0, self.v0 = pools
        self.k, self.v, self.dpages = dev(self.k0), dev(self.v0), dev(self.pages)

    def args(self):
        return (si_amd.ptr(self.k), si_amd.ptr(self.v), self.npages, self.ps,
                si_amd.ptr(self.dpages), self.max_pages)

    def s(self):
        return ctypes.byref(self.shape)

    def rows(self, pool, seq, pos, is_k):
        return ref.rows(pool, self.pages[seq], pos, self.kv, self.D, self.ps, is_k)

    def check_pools(self, written):
        """Pools equal the old ones but for the given rows {(seq, pos): (k, v)}, whose values
        are as given; returns nothing."""
        k, v = host(self.k), host(self.v)
        for pool, old, is_k in ((k, self.k0, True), (v, self.v0, False)):
            for seq in range(len(self.pages)):
                pos = np.arange(self.max_pages * self.ps)
                now, was = (self.rows(p, seq, pos, is_k) for p in (pool, old))
                for p in pos:
                    want = written.get((seq, p))
                    want = was[p] if want is None else want[0 if is_k else 1]
                    assert np.array_equal(now[p], want, equal_nan=True), (is_k, seq, p)
            spare = np.setdiff1d(np.arange(self.npages), self.pages)
            assert np.array_equal(pool[spare], old[spare])

    def read(self, n, pos0, step, ctx):
        torch = _torch()
        kvd = self.kv * self.D
        k, v = (torch.full((n, kvd), 7.0, dtype=torch.float16, device="cuda") for _ in "kv")
        si_amd.call("si_kv4_read", self.s(), *self.args(), n, pos0, step, si_amd.ptr(ctx),
                    si_amd.ptr(k), si_amd.ptr(v), None)
        return host(k), host(v)


def _tables(npos, D):
    c, s = np.empty((npos, D // 2), np.float32), np.empty((npos, D // 2), np.float32)
    si_amd.call("si_rope_table", npos, D, 1e6, si_amd.ptr(c), si_amd.ptr(s))
    return c, s


def _rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x *= np.exp(rng.normal(0, 1, width)).astype(np.float32)
    return x


def _append(c, qkv, ld, n, pos0, step, max_pos, ctx, tab):
    q = zeros(n * c.q * c.D, _torch().float32)
    si_amd.call("si_rope_kv4_append", c.s(), si_amd.ptr(qkv), ld, n, pos0, step, max_pos,
                si_amd.ptr(ctx), si_amd.ptr(tab[0]), si_amd.ptr(tab[1]), si_amd.ptr(q), *c.args(),
                None)
    return host(q).reshape(n, c.q, c.D)


def _rope32(x, pos, tab):
    """fp32 operation by operation, as the reference's rope rounds."""
    H = x.shape[2] // 2
    cs, sn = tab[0][pos][:, None], tab[1][pos][:, None]
    a, b = x[..., :H], x[..., H:]
    f = np.float32
    return np.concatenate([(a * cs).astype(f) - (b * sn).astype(f),
                           (b * cs).astype(f) + (a * sn).astype(f)], -1)


def _expect(c, qkv, pos, tab):
    x = qkv[:, :(c.q + 2 * c.kv) * c.D].reshape(len(qkv), -1, c.D)
    y = _rope32(x, pos, tab)
    return y[:, :c.q], ref.held(y[:, c.q:c.q + c.kv]), ref.held(x[:, c.q + c.kv:])


@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("name", NAMES)
def test_append_batch(name, ps):
    """A token a sequence, at page and unit borders; rows that are skipped; a row stride of its
    own; values that are zero, tied, subnormal, large, infinite or NaN."""
    rng = np.random.default_rng(ps + len(name))
    ctx = np.array([1, 8, 9, 16, 17, 31, 65, 70, 0, -3, 200, 2 ** 31 - 1], np.int32)
    longest, n = 70, 12
    c = Cache(rng, name, n, longest, ps, fill=False)
    tab = _tables(longest, c.D)
    ld = (c.q + 2 * c.kv) * c.D + 5
    qkv = _rows(rng, n, ld)
    v = qkv[:, (c.q + c.kv) * c.D:(c.q + 2 * c.kv) * c.D]
    v[0, :32] = 0
    v[1, :32] = 1.5
    v[1, 3] = -1.5
    v[2, :32] *= 1e-8
    v[3, :32] = rng.integers(-16, 17, 32) / 2  # values on borders
    v[4, 0:4] = [1e30, -np.inf, np.nan, 3]
    v[5, 1] = np.nan
    v[6, :32] = 1e-41
    q = _append(c, dev(qkv), ld, n, 0, 0, longest, dev(ctx), [dev(t) for t in tab])
    live = np.flatnonzero((ctx >= 1) & (ctx <= longest))
    wq, wk, wv = _expect(c, qkv[live], ctx[live] - 1, tab)
    assert np.array_equal(q[live], wq)
    assert not q[np.setdiff1d(np.arange(n), live)].any()  # skipped rows stay as they were
    c.check_pools({(i, ctx[i] - 1): (wk[j], wv[j]) for j, i in enumerate(live)})
    k16, v16 = c.read(n, 0, 0, dev(ctx))
    assert np.array_equal(k16[live].astype(np.float64), wk.reshape(len(live), -1))
    assert np.array_equal(v16[live].astype(np.float64), wv.reshape(len(live), -1))
    dead = np.flatnonzero((ctx < 1) | (ctx > c.max_pages * ps))
    assert (k16[dead] == 7).all() and (v16[dead] == 7).all()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("ps,pos0,n", [(16, 0, 1), (16, 3, 2), (16, 7, 50), (32, 8, 64),
                                       (64, 61, 67), (128, 0, 128)])
def test_append_prompt(name, ps, pos0, n):
    rng = np.random.default_rng(n + pos0)
    c = Cache(rng, name, 1, pos0 + n, ps)
    tab = _tables(pos0 + n, c.D)
    ld = (c.q + 2 * c.kv) * c.D
    qkv = _rows(rng, n, ld)
    pos = np.arange(pos0, pos0 + n)
    q = _append(c, dev(qkv), ld, n, pos0, 1, pos0 + n, None, [dev(t) for t in tab])
    wq, wk, wv = _expect(c, qkv, pos, tab)
    assert np.array_equal(q, wq)
    c.check_pools({(0, p): (wk[j], wv[j]) for j, p in enumerate(pos)})


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("step", [0, 1])
def test_write_and_read(name, step):
    """fp16 rows in and out: out equals what the rule holds, twice over (rows that were held
    once are held exactly)."""
    rng = np.random.default_rng(17 + step)
    n, pos0 = 45, 11
    c = Cache(rng, name, 1 if step else n, pos0 + n, 16, fill=False)
    ctx = None if step else rng.integers(1, pos0 + n, n).astype(np.int32)
    x = [(_rows(rng, n, c.kv * c.D) * s).astype(np.float16) for s in (3, 500)]
    x[1][5, 7], x[1][6, 1] = np.inf, np.nan
    dctx = None if step else dev(ctx)
    with np.errstate(all="ignore"):
        want = [ref.held(a.reshape(n, c.kv, c.D)) for a in x]
    for again in (0, 1):
        k, v = (dev(a.view(np.int16)) for a in x)
        si_amd.call("si_kv4_write", c.s(), si_amd.ptr(k), si_amd.ptr(v), n, pos0, step,
                    si_amd.ptr(dctx), *c.args(), None)
        pos = np.arange(pos0, pos0 + n) if step else ctx - 1
        if not again:
            c.check_pools({(0 if step else j, p): (want[0][j], want[1][j])
                           for j, p in enumerate(pos)})
        x = c.read(n, pos0, step, dctx)
        for a, w in zip(x, want):
            assert np.array_equal(a.astype(np.float64), w.reshape(n, -1))


def test_every_scale_and_border():
    """All 7-bit scales of either sign over fp16's range, with values on and next to every
    border (half steps of the scale, one ulp to either side)."""
    rng = np.random.default_rng(3)
    c = Cache(rng, "g1_d32", 1, 4096, 64)
    e, man = np.meshgrid(np.arange(-20, 10), np.arange(64, 128))
    h = np.ldexp(man / 64.0, e).ravel()
    h = h[(h <= 508) & (h * 2.0 ** 24 == np.rint(h * 2.0 ** 24))]
    h = np.concatenate([h, -h])[:, None]
    steps = np.concatenate([np.arange(-8, 8) + 0.5, np.arange(-7.5, 7.5)])[:31]
    x = np.concatenate([-128 * h, steps * 16 * h], 1).astype(np.float32)
    x = np.stack([x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(-np.inf))], 1)
    x[:, :, 0] = -128 * h  # the value that sets the scale
    x = x.reshape(-1, 32)
    x = np.resize(x, (-(-len(x) // 32768) * 32768, 32)).astype(np.float32)
    tab = [np.ones((4096, 16), np.float32), np.zeros((4096, 16), np.float32)]
    dt = [dev(t) for t in tab]
    for part in x.reshape(-1, 4096, 8, 32):
        qkv = np.concatenate([part, part, part], 1).reshape(4096, -1)
        _append(c, dev(qkv), qkv.shape[1], 4096, 0, 1, 4096, None, dt)
        k16, v16 = c.read(4096, 0, 1, None)
        want = ref.held(part).reshape(4096, -1)
        assert np.array_equal(k16.astype(np.float64), want)
        assert np.array_equal(v16.astype(np.float64), want)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention(c, q, nq, ctx, ctx0, step, max_ctx, q8=True, stream=None):
    torch = _torch()
    qd = c.q * c.D
    out = torch.full((nq, qd), 7.0, device="cuda")
    qs, d = zeros((nq, qd), torch.int8), zeros((nq, qd // 32), torch.int16)
    bs = zeros((nq, qd // 32), torch.int16)
    need = si_amd.lib().si_attention_kv4_workspace(c.s(), nq, step, max_ctx)
    ws = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    si_amd.call("si_attention_kv4", c.s(), si_amd.ptr(q), nq, *c.args(), si_amd.ptr(ctx), ctx0,
                step, max_ctx, si_amd.ptr(out), si_amd.ptr(qs) if q8 else None,
                si_amd.ptr(d) if q8 else None, si_amd.ptr(bs) if q8 else None, si_amd.ptr(ws),
                need, stream)
    torch.cuda.synchronize()
    got = host(out)
    if q8:  # the Q8_0 of the output, as si_quantize_q8_rows gives it
        wq, wd, wb = (torch.empty_like(t) for t in (qs, d, bs))
        si_amd.call("si_quantize_q8_rows", si_amd.ptr(out), nq, qd, si_amd.ptr(wq),
                    si_amd.ptr(wd), si_amd.ptr(wb), None)
        torch.cuda.synchronize()
        for a, b in ((qs, wq), (d, wd), (bs, wb)):
            assert torch.equal(a, b)
    return got.reshape(nq, c.q, c.D)


def _close(got, want, what):
    big = np.abs(want).max(axis=(-1, -2), keepdims=True)
    err = np.abs(got - want)
    assert np.isfinite(got).all(), what
    assert (err <= 2e-5 * big + 1e-30).all(), (what, float((err / (big + 1e-30)).max()))


def _want(c, q, seqs, ctxs):
    out = np.empty((len(ctxs), c.q, c.D))
    for i, (s, n) in enumerate(zip(seqs, ctxs)):
        pos = np.arange(max(n, 0))
        out[i] = ref.attend(q[i], c.rows(c.k0, s, pos, True), c.rows(c.v0, s, pos, False))
    return out


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("ps", [16, 32, 128])
def test_attention_ragged(name, ps):
    """Contexts at every border, none at all, and above max_ctx; pages in any order."""
    rng = np.random.default_rng(ps)
    ctx = np.array([1, 0, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255,
                    256, 257, 300, -5, 400], np.int32)
    longest = 300
    c = Cache(rng, name, len(ctx), longest, ps)
    q = rng.standard_normal((len(ctx), c.q, c.D)).astype(np.float32) * 2
    got = _attention(c, dev(q), len(ctx), dev(ctx), 0, 0, longest)
    _close(got, _want(c, q, range(len(ctx)), np.minimum(ctx, longest)), name)
    assert not got[1].any() and not got[-2].any()  # no context: zeros


@pytest.mark.parametrize("name", ["g7_d128", "g16_d64", "g1_d32"])
@pytest.mark.parametrize("nq,n", [(1, 1), (1, 1000), (1, 5000), (3, 2500), (70, 333)])
def test_attention_sizes(name, nq, n):
    """One context for every query (ctx_dev NULL): the splits of a long axis, and many rows."""
    rng = np.random.default_rng(n)
    c = Cache(rng, name, nq, n, 64)
    q = rng.standard_normal((nq, c.q, c.D)).astype(np.float32)
    got = _attention(c, dev(q), nq, None, n, 0, n)
    _close(got, _want(c, q, range(nq), [n] * nq), name)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("first,n", [(0, 1), (0, 2), (0, 77), (100, 1), (333, 3), (65, 130)])
def test_attention_prompt(name, first, n):
    rng = np.random.default_rng(first + n)
    c = Cache(rng, name, 1, first + n, 16)
    q = rng.standard_normal((n, c.q, c.D)).astype(np.float32)
    got = _attention(c, dev(q), n, None, first + 1, 1, first + n)
    _close(got, _want(c, q, [0] * n, np.arange(first + 1, first + n + 1)), name)


@pytest.mark.parametrize("name", ["g7_d64", "g7_d128", "g16_d64", "g3_d96"])
def test_unused_positions_may_hold_anything(name):
    """Bytes past a context (NaN and infinite scales among them) change nothing."""
    rng = np.random.default_rng(9)
    ctx = np.array([1, 5, 16, 37, 63, 100], np.int32)
    c = Cache(rng, name, len(ctx), 128, 64)
    q = dev(rng.standard_normal((len(ctx), c.q, c.D)).astype(np.float32))
    a = _attention(c, q, len(ctx), dev(ctx), 0, 0, 128)
    hb = c.ps * c.D // 2
    for i, n in enumerate(ctx):
        for p in range(n, 128):
            pg, r = c.pages[i, p // 64], p % 64
            for b in range(c.D // 32):
                at = ref._scale_byte(c.D, 64, r, b)
                for pool in (c.k0, c.v0):
                    pool[pg, :, at] = 0xff
                    pool[pg, :, at + 1] = 0x7f if p % 2 else 0x7c
    assert hb
    c.k, c.v = dev(c.k0), dev(c.v0)
    b = _attention(c, q, len(ctx), dev(ctx), 0, 0, 128)
    assert np.array_equal(a, b)


def test_attention_extremes():
    """Scores far apart, equal values, a scale of zero, values at both ends of fp16."""
    rng = np.random.default_rng(4)
    for name in ("g7_d128", "g16_d64"):
        c = Cache(rng, name, 4, 500, 16)
        x = rng.standard_normal((c.npages * 16, c.kv, c.D)).astype(np.float32)
        for i, f in enumerate((2e4, 1e-6, 0.0, 1.0)):  # V's size, a sequence each
            for pg in c.pages[i]:
                x[pg * 16:pg * 16 + 16] = x[pg * 16:pg * 16 + 16] * f
        c.v0 = ref.pack(x, c.kv, c.D, 16, False)
        c.v = dev(c.v0)
        q = rng.standard_normal((4, c.q, c.D)).astype(np.float32)
        q[3] *= 40  # one weight takes all
        got = _attention(c, dev(q), 4, None, 500, 0, 500)
        want = _want(c, q, range(4), [500] * 4)
        assert not got[2].any()
        # q * 40: scores of some hundreds, whose fp32 rounding (2^-24 * 500 * log2 e
        # * a few) moves a weight by 2e-4
        big = np.abs(want).max(axis=(1, 2), keepdims=True)
        tol = np.array([2e-5, 2e-5, 2e-5, 4e-4])[:, None, None]
        assert (np.abs(got - want) <= tol * big + 1e-30).all()


def test_bad_page_ids_stay_inside():
    """Ids outside the pool are clamped: the result is that of the clamped list."""
    rng = np.random.default_rng(8)
    c = Cache(rng, "g7_d128", 2, 100, 16)
    c.pages[0, 2], c.pages[1, 3] = -7, 1 << 30
    c.dpages = dev(c.pages)
    q = rng.standard_normal((2, c.q, c.D)).astype(np.float32)
    got = _attention(c, dev(q), 2, None, 100, 0, 100)
    c.pages = np.clip(c.pages, 0, c.npages - 1)
    _close(got, _want(c, q, range(2), [100, 100]), "clamped")


def test_attention_repeats_its_bits():
    """Same inputs, same bits: on another stream, and replayed from a graph between other work."""
    torch = _torch()
    rng = np.random.default_rng(2)
    c = Cache(rng, "g7_d128", 9, 900, 64)
    ctx = dev(rng.integers(0, 901, 9).astype(np.int32))
    q = dev(rng.standard_normal((9, c.q, c.D)).astype(np.float32))
    a = _attention(c, q, 9, ctx, 0, 0, 900)
    st = torch.cuda.Stream()
    b = _attention(c, q, 9, ctx, 0, 0, 900, stream=ctypes.c_void_p(st.cuda_stream))
    assert np.array_equal(a, b)
    out = torch.zeros(9, c.q * c.D, device="cuda")
    need = si_amd.lib().si_attention_kv4_workspace(c.s(), 9, 0, 900)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        si_amd.call("si_attention_kv4", c.s(), si_amd.ptr(q), 9, *c.args(), si_amd.ptr(ctx), 0, 0,
                    900, si_amd.ptr(out), None, None, None, si_amd.ptr(ws), need,
                    si_amd.stream_handle())
    for _ in range(3):
        out.zero_()
        ws.fill_(255)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(out).reshape(a.shape), a)


# ---------------------------------------------------------------------------
# page copies
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("npools,page_bytes,npages,n", [
    (1, 4096, 5, 1), (56, 1152, 40, 7), (3, 18432, 30, 15), (65, 64, 1000, 500), (2, 20, 9, 4),
    (1, 7, 12, 5), (2, 65536, 12, 6), (1, 16, 900, 450),
    (2, 1000016, 150, 70), (2, 65536, 2100, 1024), (1, 2000001, 140, 70)])  # past 256 MB
def test_copy_pages(npools, page_bytes, npages, n):
    torch = _torch()
    rng = np.random.default_rng(n)
    old = rng.integers(0, 256, (npools, npages, page_bytes), dtype=np.uint8)
    pools = dev(old)
    dst = rng.permutation(npages)[:n].astype(np.int32)
    rest = np.setdiff1d(np.arange(npages), dst)
    src = rng.choice(rest, n).astype(np.int32)  # a page may be read many times
    addr = (ctypes.c_void_p * npools)(*(pools[i].data_ptr() for i in range(npools)))
    si_amd.call("si_kv_copy_pages", addr, npools, page_bytes, npages, si_amd.ptr(src),
                si_amd.ptr(dst), n, None)
    torch.cuda.synchronize()
    want = old.copy()
    want[:, dst] = old[:, src]
    assert np.array_equal(host(pools), want)


def test_copy_pages_captured():
    """The graph holds its own lists."""
    torch = _torch()
    pools = torch.arange(2 * 6 * 64, dtype=torch.int32, device="cuda").view(2, 6, 64)
    want = pools.clone()
    want[:, 4], want[:, 5] = want[:, 0], want[:, 1]
    addr = (ctypes.c_void_p * 2)(*(p.data_ptr() for p in pools))
    src, dst = np.array([0, 1], np.int32), np.array([4, 5], np.int32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        si_amd.call("si_kv_copy_pages", addr, 2, 256, 6, si_amd.ptr(src), si_amd.ptr(dst), 2,
                    si_amd.stream_handle())
    src[:], dst[:], addr[0] = 2, 3, None
    for _ in range(3):
        pools[:, 4:].zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(pools, want)


@pytest.mark.parametrize("name", ["g7_d128", "g16_d64"])
def test_bad_heads_stay_alone(name):
    """NaN, infinities and sizes far apart in one query head leave the other heads' bits."""
    rng = np.random.default_rng(6)
    c = Cache(rng, name, 3, 700, 64)
    q = rng.standard_normal((3, c.q, c.D)).astype(np.float32)
    a = _attention(c, dev(q), 3, None, 700, 0, 700)
    for bad in (np.nan, np.inf, 1e30, 1e-30):
        q2 = q.copy()
        q2[1, 3] *= np.float32(bad)
        b = _attention(c, dev(q2), 3, None, 700, 0, 700, q8=False)
        keep = np.ones((3, c.q), bool)
        keep[1, 3] = False
        assert np.array_equal(a[keep], b[keep]), bad
        if np.isnan(bad):
            assert np.isnan(b[1, 3]).all()
        if bad in (1e30, 1e-30):  # one weight takes all; all weights are equal
            k, v = (c.rows(p, 1, np.arange(700), i) for p, i in ((c.k0, True), (c.v0, False)))
            want = ref.attend(q2[1], k, v)[3]
            assert np.abs(b[1, 3] - want).max() <= 2e-5 * np.abs(want).max()


def test_large_scores_keep_their_differences():
    """Scores of 2^14 and weights that differ in all their bits: the weights' error goes with the
    differences of the scores (as a difference of rounded scores it would be 2^14 2^-24 = 1e-3)."""
    rng = np.random.default_rng(12)
    for name in ("g7_d128", "g16_d64"):
        c = Cache(rng, name, 2, 600, 64)
        x = np.zeros((c.npages * 64, c.kv, c.D), np.float32)
        x[:, :, 0] = 8.0  # the block's scale, 1: values are whole numbers
        x[:, :, 1:32] = rng.integers(0, 2, (len(x), c.kv, 31))
        c.k0 = ref.pack(-x, c.kv, c.D, 64, True)
        c.k = dev(c.k0)
        q = np.zeros((2, c.q, c.D), np.float32)
        q[:, :, 0] = -2.0 ** 14  # times -8 over sqrt(D): the same large score for every position
        q[:, :, 1:32] = rng.integers(-8, 9, (2, c.q, 31))
        got = _attention(c, dev(q), 2, None, 600, 0, 600)
        _close(got, _want(c, q, range(2), [600] * 2), name)


@pytest.mark.parametrize("name,n,first", [
    ("g7_d128", 321, 40), ("g7_d128", 322, 40), ("g1_d32", 1125, 0), ("g1_d32", 1126, 0),
    ("g16_d128", 562, 3), ("g16_d128", 563, 3), ("g9_d32", 50, 2500), ("g7_d64", 7, 4000),
    ("g3_d96", 17, 1203), ("g16_d64", 90, 1000), ("g8_d96", 33, 15)])
def test_prompts_both_ways(name, n, first):
    """Over the pages in blocks of 16 rows (split or not) and, past 9000 rows, by fp16 rows: the
    first, the last and some queries between against 64 bits, and all against each query alone."""
    rng = np.random.default_rng(n)
    c = Cache(rng, name, 1, first + n, 32)
    q = rng.standard_normal((n, c.q, c.D)).astype(np.float32)
    got = _attention(c, dev(q), n, None, first + 1, 1, first + n)
    some = sorted({0, 1, n // 3, n // 2, n - 2, n - 1})
    _close(got[some], _want(c, q[some], [0] * len(some), first + 1 + np.array(some)), name)
    for i in range(0, n, 41):
        one = _attention(c, dev(q[i:i + 1]), 1, None, first + 1 + i, 0, first + n)
        _close(got[i:i + 1], one.astype(np.float64), (name, i))


@pytest.mark.parametrize("name,nq,longest", [
    ("g7_d128", 1, 640), ("g7_d128", 1, 641), ("g7_d128", 49, 1500), ("g7_d128", 64, 2047),
    ("g7_d128", 65, 1700), ("g7_d64", 97, 2000), ("g16_d64", 128, 1900), ("g16_d64", 300, 300),
    ("g3_d96", 30, 1801), ("g3_d96", 96, 33), ("g1_d32", 32, 2000), ("g1_d32", 25, 4096),
    ("g16_d128", 193, 1500), ("g16_d128", 70, 3000), ("g9_d32", 200, 1700),
    ("g7_d128", 1, 512), ("g7_d128", 1, 768), ("g7_d128", 1, 769), ("g7_d64", 1, 1024),
    ("g7_d64", 1, 1025), ("g3_d96", 4, 1280), ("g3_d96", 4, 1281), ("g1_d32", 3, 1984),
    ("g16_d128", 256, 700), ("g16_d128", 257, 700), ("g8_d96", 20, 1400),
    ("g7_d128", 76, 2000), ("g7_d128", 77, 2000), ("g3_d96", 39, 1950), ("g1_d32", 65, 2750),
    ("g1_d32", 160, 700), ("g16_d64", 205, 2300)])
def test_every_plan(name, nq, longest):
    """Calls on both sides of the rules that choose workgroups and chunks, with contexts from
    none to the longest: a few rows against 64 bits, all of them against calls of one query
    (another plan: fp32 sums in another order)."""
    rng = np.random.default_rng(nq)
    c = Cache(rng, name, nq, longest, 64)
    ctx = rng.integers(0, longest + 1, nq).astype(np.int32)
    ctx[rng.integers(0, nq)] = longest
    q = rng.standard_normal((nq, c.q, c.D)).astype(np.float32)
    got = _attention(c, dev(q), nq, dev(ctx), 0, 0, longest)
    some = sorted({0, nq - 1, int(ctx.argmax()), int(ctx.argmin())})
    _close(got[some], _want(c, q[some], some, ctx[some]), name)
    equal = _attention(c, dev(q), nq, None, longest, 0, longest)  # contexts from the host
    _close(equal[some], _want(c, q[some], some, [longest] * len(some)), name)
    pages = c.dpages
    for i in range(0, nq, 7):
        c.dpages = pages[i:i + 1]
        one = _attention(c, dev(q[i:i + 1]), 1, dev(ctx[i:i + 1]), 0, 0, longest)
        _close(got[i:i + 1], one.astype(np.float64), (name, i))


@pytest.mark.parametrize("name", ["g7_d128", "g9_d32", "g1_d32"])
@pytest.mark.parametrize("big", [1e34, 1e38, 3.4e38])
def test_largest_queries(name, big):
    """Queries up to fp32's largest: every weight 0 or 1 (the two best scores of 40 differ by far
    more than a rounding of either), which no unit's overflow may turn into NaN."""
    rng = np.random.default_rng(5)
    c = Cache(rng, name, 3, 300, 32)
    q = (np.clip(rng.standard_normal((3, c.q, c.D)), -1, 1) * big).astype(np.float32)
    for ctx in (40, 300):
        got = _attention(c, dev(q), 3, None, ctx, 0, 300)
        _close(got, _want(c, q, range(3), np.full(3, ctx)), (name, big, ctx))
    got = _attention(c, dev(q), 3, None, 38, 1, 300)
    _close(got, _want(c, q, [0] * 3, np.arange(38, 41)), (name, big))


def test_prompts_of_a_very_long_cache():
    """More rows than go over the pages, in lists of 2^27 positions: no fp16 rows of them all."""
    rng = np.random.default_rng(6)
    c = Cache(rng, "g1_d32", 1, 2048, 2048)
    n, first = 1200, 7
    q = rng.standard_normal((n, c.q, c.D)).astype(np.float32)
    some = np.array([0, 1, 600, n - 1])
    want = _want(c, q[some], [0] * len(some), first + some)
    by_rows = _attention(c, dev(q), n, None, first, 1, 2048)
    _close(by_rows[some], want, "rows")
    c.max_pages = (1 << 27) // 2048
    c.dpages = dev(np.full((1, c.max_pages), c.pages[0, 0], np.int32))
    ws = si_amd.lib().si_attention_kv4_workspace(c.s(), n, 1, 1 << 27)
    assert ws < 1 << 28
    _close(_attention(c, dev(q), n, None, first, 1, 1 << 27)[some], want, "pages")


def test_pools_past_4_gib():
    """Pages more than 2^32 bytes into their pools: written, read, attended to and copied; and a
    prompt whose fp16 rows of max_ctx positions take 8 GiB of workspace."""
    torch = _torch()
    rng = np.random.default_rng(9)
    q, kv, D = SHAPES["g1_d32"]
    ps, npages, n = 65536, 480, 66000
    shape = si_amd.make_shape(32, q, kv, D)
    s = ctypes.byref(shape)
    page = si_amd.lib().si_kv4_page_bytes(s, ps)
    pools = [torch.empty(npages * page, dtype=torch.uint8, device="cuda") for _ in "kv"]
    assert pools[0].numel() > 1 << 32
    x = [rng.standard_normal((n, kv, D)).astype(np.float16) for _ in "kv"]
    held = [ref.held(t.astype(np.float32)) for t in x]
    dx = [dev(t) for t in x]
    lists = dev(np.array([[479, 470], [3, 478]], np.int32))

    def cache(seq):
        return (si_amd.ptr(pools[0]), si_amd.ptr(pools[1]), npages, ps, si_amd.ptr(lists[seq]), 2)

    def rows(seq, first, count):
        out = [torch.empty(count, kv, D, dtype=torch.float16, device="cuda") for _ in "kv"]
        si_amd.call("si_kv4_read", s, *cache(seq), count, first, 1, None, si_amd.ptr(out[0]),
                    si_amd.ptr(out[1]), None)
        return [host(t).astype(np.float64) for t in out]

    si_amd.call("si_kv4_write", s, si_amd.ptr(dx[0]), si_amd.ptr(dx[1]), n, 0, 1, None, *cache(0),
                None)
    addr = (ctypes.c_void_p * 2)(*(t.data_ptr() for t in pools))
    src, dst = np.array([479, 470], np.int32), np.array([3, 478], np.int32)
    si_amd.call("si_kv_copy_pages", addr, 2, page, npages, si_amd.ptr(src), si_amd.ptr(dst), 2, None)
    qs = rng.standard_normal((3, q, D)).astype(np.float32)
    want = np.stack([ref.attend(qs[i], held[0][:n - 2 + i], held[1][:n - 2 + i])
                     for i in range(3)])
    for seq in (0, 1):
        for got, w in zip(rows(seq, 0, n), held):
            assert np.array_equal(got, w)
        need = si_amd.lib().si_attention_kv4_workspace(s, 3, 1, n)
        ws, out = empty((max(need, 1),), torch.uint8), empty((3, q, D), torch.float32)
        si_amd.call("si_attention_kv4", s, si_amd.ptr(dev(qs)), 3, *cache(seq), None, n - 2, 1, n,
                    si_amd.ptr(out), None, None, None, si_amd.ptr(ws), need, None)
        _close(host(out), want, seq)
    nq, max_ctx = 1130, 1 << 23
    long_list = dev(np.full((1, max_ctx // ps), 479, np.int32))
    need = si_amd.lib().si_attention_kv4_workspace(s, nq, 1, max_ctx)
    assert need == max_ctx * kv * D * 4
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    q2 = dev(np.repeat(qs[:1], nq, 0))
    out = empty((nq, q, D), torch.float32)
    si_amd.call("si_attention_kv4", s, si_amd.ptr(q2), nq, si_amd.ptr(pools[0]),
                si_amd.ptr(pools[1]), npages, ps, si_amd.ptr(long_list), max_ctx // ps, None, 1, 1,
                max_ctx, si_amd.ptr(out), None, None, None, si_amd.ptr(ws), need, None)
    some = np.array([0, 1, 700, nq - 1])
    _close(host(out)[some], np.stack([ref.attend(qs[0], held[0][:i + 1], held[1][:i + 1])
                                      for i in some]), "rows")


def test_attention_captured_and_on_a_stream():
    """Split calls of ragged batches: two captured graphs that share a workspace, replayed in turn
    with contexts and queries changed between and eager calls beside, and a call on a stream of the
    caller's, give the eager bits."""
    torch = _torch()
    rng = np.random.default_rng(12)
    nq, longest = 20, 3000
    c = Cache(rng, "g7_d128", nq, longest, 64)
    need = si_amd.lib().si_attention_kv4_workspace(c.s(), nq, 0, longest)
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    sets = []
    for i in range(2):
        sets.append([torch.zeros(nq, c.q, c.D, device="cuda"),
                     torch.ones(nq, dtype=torch.int32, device="cuda"),
                     torch.empty(nq, c.q, c.D, device="cuda")])

    def call(q, ctx, out, stream=None):
        si_amd.call("si_attention_kv4", c.s(), si_amd.ptr(q), nq, *c.args(), si_amd.ptr(ctx), 0, 0,
                    longest, si_amd.ptr(out), None, None, None, si_amd.ptr(ws), need,
                    si_amd.stream_handle(stream))

    graphs = []
    for s in sets:
        call(*s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(*s)
        graphs.append(g)
    side = torch.cuda.Stream()
    for turn in range(4):
        for s, g in zip(sets, graphs):
            s[0].copy_(dev(rng.standard_normal((nq, c.q, c.D)).astype(np.float32)))
            ctx = rng.integers(0, longest + 1, nq).astype(np.int32)
            if turn == 1:
                ctx[:] = longest
            s[1].copy_(dev(ctx))
            call(*s)
            torch.cuda.synchronize()
            want = s[2].clone()
            s[2].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(s[2], want), turn
            s[2].zero_()
            side.wait_stream(torch.cuda.current_stream())
            call(*s, side)
            side.synchronize()
            assert torch.equal(s[2], want), turn
    some = [0, 7, nq - 1]
    _close(host(want)[some], _want(c, host(s[0])[some], some, ctx[some]), "last")
