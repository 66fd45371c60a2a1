"""A layer and a decode stack over 4-bit K/V pages (si_layer_decode_kv4,
si_stack_create_kv), forks and compaction included.

The layer, stage by stage on its own intermediates: the q|k|v rows rotated and held
as tests/kv4_ref.py says, bit for bit; attention over the pages as they now are
(2e-5 of a row's largest value, as tests/test_gpu_kv4.py derives); everything after
it the library's other calls on the same inputs, bit for bit (SI_LAYER_EXACT).

The stack: the same bits as its layers driven one by one over pools of the test's
own, for sequences that join, fork, are cut back, leave, and are compacted."""
import ctypes

import numpy as np
import pytest

import si_amd
from oracle.oracle_py import make_shape as or_shape
from tests import kv4_ref as ref
from tests.gpu_helpers import dev, device_view, empty, host, make_layer
from tests.test_gpu_kv4 import _close, _rope32, _tables

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def _buf(L, name, rows, n, dtype=None):
    t = device_view(L.buffer(name), rows * n, dtype or _torch().float32)
    return t.clone().view(rows, n)


def _weights(L, which):
    qs, d, tile, n, k = L.weights(which)
    return qs, d, tile, n, k


def _gemm(w, xq, xd, m, residual=None):
    torch = _torch()
    qs, d, tile, n, k = w
    out = torch.empty(m, n, device="cuda")
    if m == 1:
        sums = xq.view(-1, 32).to(torch.int32).sum(1).to(torch.int16)
        si_amd.call("si_matvec_q4q8", qs, d, tile, n, k, si_amd.ptr(xq), si_amd.ptr(xd),
                    si_amd.ptr(sums), None, si_amd.ptr(residual), si_amd.ptr(out), 1, None)
    else:
        si_amd.call("si_gemm_q4q8", qs, d, tile, n, k, si_amd.ptr(xq), si_amd.ptr(xd), m, None,
                    si_amd.ptr(residual), si_amd.ptr(out), n, si_amd.SI_GEMM_EXACT, None, 0, None)
    return out


@pytest.mark.parametrize("model,nseq,ps", [("0.5b", 6, 16), ("0.5b", 1, 64), ("7b", 3, 64),
                                           ("0.5b", 70, 32)])
@pytest.mark.parametrize("full", [True, False])
def test_layer_stage_by_stage(oracle, model, nseq, ps, full):
    torch = _torch()
    sd = dict(si_amd.SHAPES[model])
    if not full:
        sd["ffn"] = 0
    s, os_ = si_amd.make_shape(**sd), or_shape(**sd)
    H, D, F = s.hidden, s.hdim, s.ffn
    qd = s.qheads * D
    lay = make_layer(oracle, os_, 11, ffn=full)
    rng = np.random.default_rng(nseq)
    max_ctx = 300
    ctx = rng.integers(1, max_ctx + 1, nseq).astype(np.int32)
    ctx[0], ctx[-1] = 1, max_ctx
    mp = -(-max_ctx // ps)
    npages = nseq * mp + 2
    table = rng.permutation(npages)[:nseq * mp].reshape(nseq, mp).astype(np.int32)
    kp, vp = (ref.pack(rng.standard_normal((npages * ps, s.kvheads, D)).astype(np.float32),
                       s.kvheads, D, ps, k) for k in (True, False))
    dk, dv, dt, dc = dev(kp), dev(vp), dev(table), dev(ctx)
    x = dev(rng.standard_normal((nseq, H)).astype(np.float32))
    L = si_amd.Layer(s, lay, nseq, max_ctx)
    out = empty((nseq, H), torch.float32)
    flags = si_amd.SI_LAYER_EXACT | (0 if full else si_amd.SI_LAYER_ATTN_ONLY)
    L.decode_kv4(x, nseq, dk, dv, npages, ps, dt, mp, dc, max_ctx, out, flags)
    torch.cuda.synchronize()
    qkv = host(_buf(L, "QKV", nseq, qd + 2 * s.kvheads * D)).reshape(nseq, -1, D)
    y = _rope32(qkv, ctx - 1, _tables(max_ctx, D))
    q = host(_buf(L, "Q", nseq, qd)).reshape(nseq, s.qheads, D)
    assert np.array_equal(q, y[:, :s.qheads])
    # the new rows as the rule holds them, the others as they were
    k1, v1 = host(dk), host(dv)
    want_k, want_v = ref.held(y[:, s.qheads:s.qheads + s.kvheads]), ref.held(
        qkv[:, s.qheads + s.kvheads:])
    attn = host(_buf(L, "ATTN", nseq, qd)).reshape(nseq, s.qheads, D)
    want = np.empty_like(attn, dtype=np.float64)
    for i, n in enumerate(ctx):
        pos = np.arange(n)
        rk, rv = (ref.rows(p, table[i], pos, s.kvheads, D, ps, b) for p, b in ((k1, True), (v1, False)))
        ok, ov = (ref.rows(p, table[i], pos, s.kvheads, D, ps, b) for p, b in ((kp, True), (vp, False)))
        assert np.array_equal(rk[:-1], ok[:-1]) and np.array_equal(rv[:-1], ov[:-1])
        assert np.array_equal(rk[-1], want_k[i]) and np.array_equal(rv[-1], want_v[i])
        want[i] = ref.attend(q[i], rk, rv)
    _close(attn, want, model)
    # from the attention on: the library's calls on the layer's own values
    at = _buf(L, "ATTN", nseq, qd)
    aq, ad = _buf(L, "ATTQ_QS", nseq, qd, torch.int8), _buf(L, "ATTQ_D", nseq, qd // 32, torch.int16)
    wq, wd = torch.empty_like(aq), torch.empty_like(ad)
    si_amd.call("si_quantize_q8_rows", si_amd.ptr(at), nseq, qd, si_amd.ptr(wq), si_amd.ptr(wd),
                None, None)
    torch.cuda.synchronize()
    assert torch.equal(aq, wq) and torch.equal(ad, wd)
    o = _gemm(_weights(L, 1), aq, ad, nseq)
    if not full:
        assert torch.equal(out, o)
    else:
        h, hn = torch.empty_like(x), torch.empty(nseq, H, dtype=torch.int8, device="cuda")
        hd = torch.empty(nseq, H // 32, dtype=torch.int16, device="cuda")
        gain = dev(lay["post_norm"])
        si_amd.call("si_residual_rmsnorm_q8", si_amd.ptr(x), si_amd.ptr(o), si_amd.ptr(gain), nseq,
                    H, s.rms_eps, si_amd.ptr(h), None, si_amd.ptr(hn), si_amd.ptr(hd), None, None)
        gu = _gemm(_weights(L, 2), hn, hd, nseq)
        fq = torch.empty(nseq, F, dtype=torch.int8, device="cuda")
        fd = torch.empty(nseq, F // 32, dtype=torch.int16, device="cuda")
        si_amd.call("si_swiglu_q8", si_amd.ptr(gu), nseq, F, None, si_amd.ptr(fq), si_amd.ptr(fd),
                    None, None)
        assert torch.equal(out, _gemm(_weights(L, 3), fq, fd, nseq, h))
    # the default roundings, and the operand-tiled Q8_0 that they stream: the
    # attention's copy holds the same values
    L.decode_kv4(x, nseq, dk, dv, npages, ps, dt, mp, dc, max_ctx, out,
                 0 if full else si_amd.SI_LAYER_ATTN_ONLY, capture=False)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    L.close()


def test_streamed_projection_reads_the_attention(oracle):
    """2 to 64 rows without SI_LAYER_EXACT: W_O streams the attention's operand-tiled Q8_0, so
    the layer's attn_out is si_gemm_q4q8's with SI_GEMM_TILED_A on the planar one."""
    torch = _torch()
    sd = si_amd.SHAPES["0.5b"]
    s, os_ = si_amd.make_shape(**sd), or_shape(**sd)
    lay, rng, nseq, ps = make_layer(oracle, os_, 5), np.random.default_rng(5), 33, 16
    qd, D, max_ctx = s.qheads * s.hdim, s.hdim, 400
    mp = max_ctx // ps
    table = rng.permutation(nseq * mp).reshape(nseq, mp).astype(np.int32)
    pools = [dev(ref.pack(rng.standard_normal((nseq * mp * ps, s.kvheads, D)).astype(np.float32),
                          s.kvheads, D, ps, k)) for k in (True, False)]
    ctx = dev(rng.integers(1, max_ctx + 1, nseq).astype(np.int32))
    x = dev(rng.standard_normal((nseq, s.hidden)).astype(np.float32))
    L = si_amd.Layer(s, lay, nseq, max_ctx)
    out = empty((nseq, s.hidden), torch.float32)
    L.decode_kv4(x, nseq, *pools, nseq * mp, ps, dev(table), mp, ctx, max_ctx, out)
    torch.cuda.synchronize()
    aq, ad = _buf(L, "ATTQ_QS", nseq, qd, torch.int8), _buf(L, "ATTQ_D", nseq, qd // 32, torch.int16)
    P = (nseq + 31) // 32
    tq = torch.zeros(P * 32 * qd, dtype=torch.int8, device="cuda")
    td = torch.zeros(P * qd, dtype=torch.int16, device="cuda")
    si_amd.call("si_q8_tile", si_amd.ptr(aq), si_amd.ptr(ad), nseq, qd, si_amd.ptr(tq),
                si_amd.ptr(td), None)
    qs, d, tile, n, k = L.weights(1)
    o = torch.empty(nseq, n, device="cuda")
    si_amd.call("si_gemm_q4q8", qs, d, tile, n, k, si_amd.ptr(tq), si_amd.ptr(td), nseq, None, None,
                si_amd.ptr(o), n, si_amd.SI_GEMM_TILED_A, None, 0, None)
    torch.cuda.synchronize()
    assert torch.equal(o, _buf(L, "ATTN_OUT", nseq, s.hidden))
    L.close()


def test_layer_refusals(oracle):
    sd = dict(si_amd.SHAPES["0.5b"], ffn=0)
    s = si_amd.make_shape(**sd)
    L = si_amd.Layer(s, make_layer(oracle, or_shape(**sd), 1, ffn=False), 4, 64)
    t = _torch().zeros(1 << 16, dtype=_torch().uint8, device="cuda")
    p = t.data_ptr()
    good = [L.h, p, 2, p, p, 8, 16, p, 4, None, 5, 64, p, si_amd.SI_LAYER_ATTN_ONLY, None]
    for at, bad, msg in ((1, None, b"NULL"), (12, None, b"NULL"), (13, 5, b"flags"), (2, 0, b"nseq"),
                         (2, 5, b"nseq"), (11, 65, b"max_ctx"), (11, 0, b"max_ctx"),
                         (10, 0, b"context"), (10, 65, b"context"), (3, p + 8, b"16-byte"),
                         (6, 8, b"power of two"), (8, 3, b"do not cover"), (5, 0, b">= 1"),
                         (7, None, b"NULL")):
        args = list(good)
        args[at] = bad
        assert si_amd.lib().si_layer_decode_kv4(*args) == si_amd.SI_ERR_ARG, (at, bad)
        assert msg in si_amd.lib().si_last_error(), (at, si_amd.lib().si_last_error())
    L.close()


class Mirror:
    """The stack's layers and pools again, driven call by call."""

    def __init__(self, H, st, s, lays, fmt, npages, ps, max_seqs, max_ctx):
        torch = _torch()
        self.H, self.st, self.s, self.fmt, self.npages, self.ps = H, st, s, fmt, npages, ps
        self.pages, self.max_seqs, self.mp = H.si_stack_pages(st), max_seqs, -(-max_ctx // ps)
        kvd = s.kvheads * s.hdim
        self.pb = ps * kvd * 9 // 16 if fmt else ps * kvd * 2
        if fmt:
            assert self.pb == si_amd.lib().si_kv4_page_bytes(ctypes.byref(s), ps)
        self.layers = [si_amd.Layer(s, lay, max_seqs, max_ctx) for lay in lays]
        get = (H.si_stack_k_pool, H.si_stack_v_pool)
        self.real = [[device_view(f(st, l), npages * self.pb, torch.uint8).view(npages, self.pb)
                      for f in get] for l in range(len(lays))]
        for pair in self.real:
            for t in pair:
                t.zero_()
        self.mem = [[t.clone() for t in pair] for pair in self.real]

    def table(self):
        t = np.ctypeslib.as_array(self.H.si_kv_page_table(self.pages),
                                  shape=(self.max_seqs * self.mp,))
        return t.reshape(self.max_seqs, self.mp).copy()

    def lens(self, seqs):
        return np.array([self.H.si_kv_seq_len(self.pages, i) for i in seqs], np.int32)

    def prepare(self, seqs):
        before, lens = self.table(), self.lens(seqs)
        ids = (ctypes.c_int * len(seqs))(*seqs)
        if self.H.si_stack_prepare(self.st, ids, len(seqs)) != 0:
            return False
        after, moved = self.table(), 0
        for i, n in zip(seqs, lens):
            at = n // self.ps
            if n % self.ps and before[i, at] != after[i, at]:
                moved += 1
                for pair in self.mem:
                    for t in pair:
                        t[after[i, at]] = t[before[i, at]]
        self.moved = moved
        return True

    def step(self, seqs, x):
        torch = _torch()
        n = len(seqs)
        out = empty((n, self.s.hidden), torch.float32)
        self.H.si_stack_decode(self.st, si_amd.ptr(x), si_amd.ptr(out), si_amd.SI_LAYER_FULL, None)
        tab, ctx = dev(self.table()[seqs]), dev(self.lens(seqs))
        most, cur = int(self.lens(seqs).max()), x
        for L, (k, v) in zip(self.layers, self.mem):
            o = empty((n, self.s.hidden), torch.float32)
            f = L.decode_kv4 if self.fmt else L.decode_paged
            f(cur, n, k, v, self.npages, self.ps, tab, self.mp, ctx, most, o,
              si_amd.SI_LAYER_FULL, capture=False)
            cur = o
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
        assert torch.equal(out, cur)
        return out

    def check_pools(self):
        torch = _torch()
        for real, mem in zip(self.real, self.mem):
            for a, b in zip(real, mem):
                assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", [si_amd.SI_KV_F16, si_amd.SI_KV_Q4])
def test_stack_forks_and_compacts(oracle, fmt):
    torch = _torch()
    H = si_amd.host_lib()
    sd = si_amd.SHAPES["0.5b"]
    s, os_ = si_amd.make_shape(**sd), or_shape(**sd)
    nl, max_seqs, max_ctx, ps, npages = 2, 5, 96, 16, 18
    lays = [make_layer(oracle, os_, 80 + l) for l in range(nl)]
    keep = [{k: np.ascontiguousarray(v) for k, v in t.items() if v is not None} for t in lays]
    hosts = (si_amd.LayerHost * nl)(*[si_amd.LayerHost(**{k: v.ctypes.data for k, v in kk.items()})
                                      for kk in keep])
    st = H.si_stack_create_kv(ctypes.byref(s), ctypes.cast(hosts, ctypes.c_void_p), nl, max_seqs,
                              max_ctx, npages, ps, fmt)
    M = Mirror(H, st, s, lays, fmt, npages, ps, max_seqs, max_ctx)
    pg, rng = M.pages, np.random.default_rng(7)

    def x(n):
        return dev(rng.standard_normal((n, s.hidden)).astype(np.float32))

    a, b = H.si_kv_seq_add(pg), H.si_kv_seq_add(pg)
    for _ in range(21):
        assert M.prepare([a, b])
        M.step([a, b], x(2))
    # a fork: the next step copies one page; the same token gives both the same row
    c = H.si_stack_fork(st, a)
    assert c == 2 and M.prepare([a, b, c]) and M.moved == 1
    t = x(3)
    t[2] = t[0]
    o = M.step([a, b, c], t)
    assert torch.equal(o[0], o[2]) and not torch.equal(o[0], o[1])
    for _ in range(15):  # they part, over a page border
        assert M.prepare([a, b, c]) and M.moved == 0
        o = M.step([a, b, c], x(3))
    assert not torch.equal(o[0], o[2])
    # what a and c share is one copy of it
    tab = M.table()
    assert tab[a, 0] == tab[c, 0] and tab[a, 1] != tab[c, 1]
    # cut back into the shared part, then grown: another copy
    d = H.si_stack_fork(st, c)
    H.si_kv_seq_truncate(pg, d, 9)
    H.si_kv_seq_free(pg, b)
    assert M.prepare([a, c, d]) and M.moved == 1
    M.step([a, c, d], x(3))
    M.check_pools()
    # compaction: the held pages are the first ones, and every sequence reads what it did
    before = M.table()
    lens = {i: int(H.si_kv_seq_len(pg, i)) for i in (a, c, d)}
    used = H.si_stack_compact(st)
    after = M.table()
    assert used == npages - H.si_kv_pages_free(pg)
    moves = {}
    for i, n in lens.items():
        for j in range(-(-n // ps)):
            assert after[i, j] < used
            moves[int(before[i, j])] = int(after[i, j])
    assert any(x != y for x, y in moves.items())
    for pair in M.mem:
        for m in pair:
            old = m.clone()
            for src, dst in moves.items():
                m[dst] = old[src]
    assert H.si_stack_nseq(st) == 0
    M.check_pools()
    for _ in range(4):
        assert M.prepare([a, c, d])
        M.step([a, c, d], x(3))
    M.check_pools()
    # forks until the pool is dry: nothing is lost by the step that fails
    f = H.si_stack_fork(st, a)
    seqs = [a, c, d, f]
    while True:
        lens = M.lens(seqs)
        if not M.prepare(seqs):
            assert np.array_equal(M.lens(seqs), lens) and H.si_stack_nseq(st) == 0
            break
        M.step(seqs, x(4))
    H.si_kv_seq_free(pg, d)
    assert M.prepare([a, c, f])
    M.step([a, c, f], x(3))
    H.si_stack_destroy(st)
    for L in M.layers:
        L.close()


def test_decode_captured(oracle):
    """A captured step replayed between other work gives the eager bits, contexts and page lists
    read at replay."""
    torch = _torch()
    sd = si_amd.SHAPES["0.5b"]
    s, os_ = si_amd.make_shape(**sd), or_shape(**sd)
    rng, nseq, ps, max_ctx = np.random.default_rng(3), 5, 32, 256
    mp = max_ctx // ps
    L = si_amd.Layer(s, make_layer(oracle, os_, 3), nseq, max_ctx)
    pools0 = [dev(ref.pack(rng.standard_normal((nseq * mp * ps, s.kvheads, s.hdim)).astype(
        np.float32), s.kvheads, s.hdim, ps, k)) for k in (True, False)]
    pools = [t.clone() for t in pools0]
    table = dev(rng.permutation(nseq * mp).reshape(nseq, mp).astype(np.int32))
    ctx = dev(np.full(nseq, 100, np.int32))
    x, out = dev(rng.standard_normal((nseq, s.hidden)).astype(np.float32)), empty(
        (nseq, s.hidden), torch.float32)

    def call():
        L.decode_kv4(x, nseq, *pools, nseq * mp, ps, table, mp, ctx, max_ctx, out, capture=False)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for i in range(3):
        ctx.copy_(dev(rng.integers(0, max_ctx + 1, nseq).astype(np.int32)))
        x.copy_(dev(rng.standard_normal((nseq, s.hidden)).astype(np.float32)))
        for t, t0 in zip(pools, pools0):
            t.copy_(t0)
        call()
        torch.cuda.synchronize()
        want, held = out.clone(), [t.clone() for t in pools]
        out.zero_()
        for t, t0 in zip(pools, pools0):
            t.copy_(t0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(torch.equal(a, b) for a, b in zip(pools, held))
    L.close()


def test_prompt_through_rows_then_decode(oracle):
    """A prompt in two pieces through an fp16 cache of its own, the second over the first's rows
    read back from the pages, then tokens decoded over them."""
    torch = _torch()
    sd = si_amd.SHAPES["0.5b"]
    s, os_ = si_amd.make_shape(**sd), or_shape(**sd)
    D, kvd, qd = s.hdim, s.kvheads * s.hdim, s.qheads * s.hdim
    rng, ps, mp, npages = np.random.default_rng(8), 16, 5, 9
    L = si_amd.Layer(s, make_layer(oracle, os_, 8), 32, 80)
    page = si_amd.lib().si_kv4_page_bytes(ctypes.byref(s), ps)
    pools = [torch.zeros(npages * page, dtype=torch.uint8, device="cuda") for _ in "kv"]
    table = rng.permutation(npages)[:mp].astype(np.int32)
    dt = dev(table.reshape(1, mp))
    cache = (si_amd.ptr(pools[0]), si_amd.ptr(pools[1]), npages, ps, si_amd.ptr(dt), mp)
    shape = ctypes.byref(s)

    def rows(n):
        return [ref.rows(host(t).reshape(npages, s.kvheads, -1), table, np.arange(n), s.kvheads, D,
                         ps, k) for t, k in zip(pools, (True, False))]

    done = 0
    for n in (21, 24):
        k, v = (torch.zeros(done + n, kvd, dtype=torch.float16, device="cuda") for _ in "kv")
        si_amd.call("si_kv4_read", shape, *cache, done, 0, 1, None, si_amd.ptr(k), si_amd.ptr(v),
                    None)
        torch.cuda.synchronize()
        before = rows(done)
        for t, want in zip((k, v), before):
            assert np.array_equal(host(t)[:done].reshape(want.shape), want)
        x = dev(rng.standard_normal((n, s.hidden)).astype(np.float32))
        L.prefill(x, n, done, k, v, empty((n, s.hidden), torch.float32))
        torch.cuda.synchronize()
        q = host(_buf(L, "Q", n, qd)).reshape(n, s.qheads, D)
        kk, vv = (host(t).astype(np.float64).reshape(-1, s.kvheads, D) for t in (k, v))
        want = np.stack([ref.attend(q[i], kk[:done + i + 1], vv[:done + i + 1]) for i in range(n)])
        _close(host(_buf(L, "ATTN", n, qd)).reshape(n, s.qheads, D), want, n)
        si_amd.call("si_kv4_write", shape, si_amd.ptr(k[done:]), si_amd.ptr(v[done:]), n, done, 1,
                    None, *cache, None)
        torch.cuda.synchronize()
        for now, old, t in zip(rows(done + n), before, (k, v)):
            assert np.array_equal(now[:done], old)
            assert np.array_equal(now[done:], ref.held(
                host(t)[done:].astype(np.float32).reshape(n, s.kvheads, D)))
        done += n
    for _ in range(3):
        done += 1
        x = dev(rng.standard_normal((1, s.hidden)).astype(np.float32))
        L.decode_kv4(x, 1, *pools, npages, ps, dt, mp, dev(np.array([done], np.int32)), 80,
                     empty((1, s.hidden), torch.float32))
        torch.cuda.synchronize()
        q = host(_buf(L, "Q", 1, qd)).reshape(1, s.qheads, D)
        _close(host(_buf(L, "ATTN", 1, qd)).reshape(1, s.qheads, D),
               ref.attend(q[0], *rows(done))[None], done)
    L.close()
