"""The layer over a ragged step's rows (si_layer_step): prompts, drafted and single tokens in one
call, over tables that si_kv_step made, checked as a chain (tests/chain.py); with a window, its
attention against 64 bits."""
import numpy as np
import pytest

import si_amd
from oracle.oracle_py import make_shape as or_shape
from tests import step_ref
from tests.chain import E2E_BOUND, LayerBuffers, check_row, end_to_end_report
from tests.gpu_helpers import close, dev, device_view, empty, host, make_layer, torch_cuda
from tests.test_gpu_step import Tables

pytestmark = pytest.mark.gpu


class Run:
    """A layer, its pools, and the tables of its sequences."""

    def __init__(self, oracle, model, nseq, page, max_ctx, max_rows, window, sinks, ffn=True):
        torch = torch_cuda()
        sd = dict(si_amd.SHAPES[model])
        if not ffn:
            sd["ffn"] = 0
        self.s, self.os = si_amd.make_shape(**sd), or_shape(**sd)
        self.lay = make_layer(oracle, self.os, 71, ffn=ffn)
        self.L = si_amd.Layer(self.s, self.lay, max_rows, max_ctx)
        self.max_pages, self.page, self.max_ctx = -(-max_ctx // page), page, max_ctx
        self.max_rows, self.window, self.sinks, self.nseq = max_rows, window, sinks, nseq
        self.npages = nseq * self.max_pages
        self.t = Tables(nseq, page, self.npages, self.max_pages, max_rows, window, sinks, seed=7)
        self.kvd = self.s.kvheads * self.s.hdim
        self.k, self.v = (torch.zeros(self.npages * page * self.kvd, dtype=torch.int16,
                                      device="cuda") for _ in range(2))
        self.have = np.zeros(nseq, np.int32)

    def step(self, x, add, max_new, flags, stream=None):
        """The step's outputs, its rows' (sequence, position), and the tables."""
        torch = torch_cuda()
        t, n = self.t, sum(add)
        add = np.array(add, np.int32)
        t.run(dev(self.have), dev(add))
        out = empty((self.max_rows, self.s.hidden), torch.float32)
        self.L.step(dev(x), self.nseq, self.max_rows, max_new, self.max_ctx, self.window,
                    self.sinks, t.start, t.ctx, t.pos, t.slot, self.k, self.v, self.npages,
                    self.page, t.pages, self.max_pages, out, flags, stream)
        torch.cuda.synchronize()
        assert host(t.status)[0] == 0
        self.have = self.have + add
        return host(out)[:n], list(zip(host(t.seq)[:n], host(t.pos)[:n]))

    def caches(self, i):
        """Sequence i's K and V rows, gathered from the pools, as fp16 bits."""
        rows = host(self.t.pages)[i].astype(np.int64)[:, None] * self.page + np.arange(self.page)
        rows = rows.reshape(-1)[:self.have[i]] % (self.npages * self.page)
        return tuple(host(x).view(np.uint16).reshape(-1, self.kvd)[rows] for x in (self.k, self.v))


def check_row_7b(oracle, s, lay, x, t, B, kc, vc, p, out):
    """check_row for 7B sums that are not in the oracle's order, its third link left out: W_O's
    output off by 2^-24 moves roundings of the post-norm's Q8 to the other side, each by a 127th
    of its block's largest value, and the layer's output by 1e-2 (test_oracle_sensitivity.py shows
    it on the oracle alone), so continued from the attention it is held to E2E_BOUND.  Every
    stage on its own inputs is held as closely as there."""
    H, QD, KVD, F = s.hidden, s.qheads * s.hdim, s.kvheads * s.hdim, s.ffn
    assert np.array_equal(B.normed[t], oracle.rmsnorm(x, lay["norm"]))
    q = oracle.rope(oracle.matvec(lay["wq"], B.xq[t], H, QD, lay["bq"]), s.qheads, s.hdim, p)
    k = oracle.rope(oracle.matvec(lay["wk"], B.xq[t], H, KVD, lay["bk"]), s.kvheads, s.hdim, p)
    close(B.q[t], q, 1e-5, "q")
    close(oracle.f16_to_f32(kc[p * KVD:(p + 1) * KVD]), oracle.f16_to_f32(oracle.f32_to_f16(k)),
          2e-3, "new K row")
    close(B.attn[t], oracle.attention_flash(s, B.q[t], kc, vc, p + 1), 2e-3, "attention")
    attq = oracle.quantize_q8(B.attn[t])
    assert np.array_equal(B.attq[t], attq)
    close(B.attn_out[t], oracle.matvec(lay["wo"], attq, QD, H), 1e-5, "W_O")
    close(B.h[t], x + B.attn_out[t], 1e-6, "residual")
    assert np.array_equal(B.xq2[t], oracle.quantize_q8(B.normed2[t]))
    gu = np.concatenate([oracle.matvec(lay[w], B.xq2[t], H, F) for w in ("wgate", "wup")])
    close(B.gu[t], gu, 1e-5, "gate|up")
    assert np.array_equal(B.actq[t], oracle.quantize_q8(B.act[t]))
    close(out, B.h[t] + oracle.matvec(lay["wdown"], B.actq[t], F, H), 1e-5, "down + residual")
    h = x + oracle.matvec(lay["wo"], attq, QD, H)
    xq2 = oracle.quantize_q8(oracle.rmsnorm(h, lay["post_norm"]))
    g, u = (oracle.matvec(lay[w], xq2, H, F) for w in ("wgate", "wup"))
    y = h + oracle.matvec(lay["wdown"], oracle.quantize_q8(oracle.swiglu(g, u)), F, H)
    assert end_to_end_report(out, y)["max_over_rms"] <= E2E_BOUND["7b"]


@pytest.mark.parametrize("model,flags", [
    ("0.5b", si_amd.SI_LAYER_FULL), ("0.5b", si_amd.SI_LAYER_EXACT),
    ("1.5b_ref", si_amd.SI_LAYER_ATTN_ONLY), ("7b", si_amd.SI_LAYER_FULL),
    ("7b", si_amd.SI_LAYER_EXACT)])
@pytest.mark.parametrize("room", [0, 60])
def test_step_chain(oracle, model, flags, room):
    """Two steps: a prompt's piece among others, then drafts and single tokens (up to 64 rows, and
    with `room` more of them)."""
    full = not flags & si_amd.SI_LAYER_ATTN_ONLY
    r = Run(oracle, model, 4, 16, 128, 40 + room, 2 ** 31 - 1, 0, ffn=full)
    rng = np.random.default_rng(72)
    for add, max_new in (([25, 0, 7, 1], 25), ([1, 3, 0, 5], 5)):
        x = rng.standard_normal((r.max_rows, r.s.hidden)).astype(np.float32)
        got, rows = r.step(x, add, max_new, flags)
        B = LayerBuffers(r.L, r.os, r.max_rows)
        for t, (i, p) in enumerate(rows):
            if t % 3 and p < 24:
                continue
            kc, vc = (c.reshape(-1) for c in r.caches(i))
            if model == "7b" and not flags & si_amd.SI_LAYER_EXACT:
                check_row_7b(oracle, r.os, r.lay, x[t], t, B, kc, vc, p, got[t])
                continue
            check_row(oracle, r.os, r.lay, x[t], t, B, kc, vc, 0, p, p + 1, got[t],
                      bool(flags & si_amd.SI_LAYER_EXACT), full=full)


def test_step_window(oracle):
    """A window and sinks over several steps, whose pages come back: the layer's attention of its
    own rotated q over the pages."""
    torch = torch_cuda()
    r = Run(oracle, "0.5b", 3, 8, 96, 48, 21, 3, ffn=False)
    r.npages = 18  # windows, not whole sequences
    r.t = Tables(3, 8, 18, r.max_pages, 48, 21, 3, seed=8)
    rng = np.random.default_rng(73)
    s, D = r.s, r.s.hdim
    taken = back = 0
    for add in ([40, 1, 4], [1, 30, 2], [3, 2, 1], [0, 4, 31], [1, 1, 1], [9, 0, 2]):
        x = rng.standard_normal((48, s.hidden)).astype(np.float32)
        got, rows = r.step(x, add, max(add), si_amd.SI_LAYER_ATTN_ONLY)
        q, attn = (host(device_view(r.L.buffer(n), 48 * s.qheads * D, torch.float32).clone())
                   .reshape(48, s.qheads, D) for n in ("Q", "ATTN"))
        for t, (i, p) in enumerate(rows):
            k, v = (c.view(np.float16).reshape(-1, s.kvheads, D) for c in r.caches(i))
            want, bound = step_ref.attend(q[t], k, v, int(p), 21, 3, s.qheads // s.kvheads)
            assert (np.abs(attn[t] - want) <= bound).all(), (add, t)
        taken, back = taken + host(r.t.status)[2], back + host(r.t.status)[3]
    # 54, 38 and 41 positions; what lies 21 behind 45, 38 and 39, whole pages past the first
    assert taken == 7 + 5 + 6 and back == 2 + 1 + 1


def test_step_replayed(oracle):
    """A step captured with its tables, replayed over growing sequences: every replay's outputs are
    the eager ones of another run."""
    torch = torch_cuda()
    eager, other = (Run(oracle, "0.5b", 3, 16, 128, 16, 40, 4) for _ in range(2))
    rng = np.random.default_rng(74)
    x = dev(np.zeros((16, eager.s.hidden), np.float32))
    have, add = dev(np.zeros(3, np.int32)), dev(np.zeros(3, np.int32))
    out = empty((16, eager.s.hidden), torch.float32)

    def calls():
        t = other.t
        t.run(have, add)
        other.L.step(x, 3, 16, 6, 128, 40, 4, t.start, t.ctx, t.pos, t.slot, other.k, other.v,
                     other.npages, 16, t.pages, other.max_pages, out, capture=False)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls()  # (no rows)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            calls()
    torch.cuda.synchronize()
    for step in range(6):
        n = rng.integers(0, 6, 3).astype(np.int32)
        xs = rng.standard_normal((16, eager.s.hidden)).astype(np.float32)
        have.copy_(dev(eager.have))
        add.copy_(dev(n))
        x.copy_(dev(xs))
        want, _ = eager.step(xs, n, 6, si_amd.SI_LAYER_FULL)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(out)[:n.sum()].view(np.uint32), want.view(np.uint32)), step


def test_step_refusals(oracle):
    torch = torch_cuda()
    r = Run(oracle, "0.5b", 2, 16, 64, 8, 40, 4, ffn=False)
    x, out = (empty((8, r.s.hidden), torch.float32) for _ in range(2))
    t = r.t

    def call(nseq=2, max_rows=8, max_new=4, max_ctx=64, window=40, sinks=4, start=t.start,
             k=r.k, page=16, npages=r.npages, max_pages=4, x=x, flags=si_amd.SI_LAYER_ATTN_ONLY):
        r.L.step(x, nseq, max_rows, max_new, max_ctx, window, sinks, start, t.ctx, t.pos, t.slot, k,
                 r.v, npages, page, t.pages, max_pages, out, flags)

    t.run(dev(r.have), dev(np.zeros(2, np.int32)))
    call()
    for bad in (dict(nseq=0), dict(nseq=1 << 16), dict(max_rows=0), dict(max_rows=9),
                dict(max_new=0), dict(max_ctx=0), dict(max_ctx=65), dict(window=0),
                dict(sinks=-1), dict(start=None), dict(k=None), dict(k=r.k[4:]), dict(page=12),
                dict(npages=0), dict(max_pages=3), dict(x=None), dict(flags=0),
                dict(flags=si_amd.SI_LAYER_ATTN_STANDARD)):
        with pytest.raises(si_amd.SiError):
            call(**bad)
    torch.cuda.synchronize()


def test_step_too_many_rows(oracle):
    """Rows and heads that one launch of the attention does not take are refused before anything
    runs, as si_attention_rows has it; the largest step of the same heads that fits is not."""
    torch = torch_cuda()
    sd = dict(hidden=32, qheads=256, kvheads=256, hdim=32, ffn=0)
    s, os_ = si_amd.make_shape(**sd), or_shape(**sd)
    n, page, max_pages = 65535, 16, 2
    L = si_amd.Layer(s, make_layer(oracle, os_, 5, ffn=False), n, 32)
    t = Tables(n, page, 8, max_pages, n, 32, 0)
    t.run(dev(np.zeros(n, np.int32)), dev(np.zeros(n, np.int32)))
    k, v = (torch.full((8 * page * 256 * 32,), 7, dtype=torch.int16, device="cuda")
            for _ in range(2))
    x, out = (empty((n, 32), torch.float32) for _ in range(2))
    out.fill_(7.0)

    def call(max_new):
        L.step(x, n, n, max_new, 32, 32, 0, t.start, t.ctx, t.pos, t.slot, k, v, 8, page, t.pages,
               max_pages, out, si_amd.SI_LAYER_ATTN_ONLY)

    with pytest.raises(si_amd.SiError, match="too many"):
        call(65)
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    call(1)
    torch.cuda.synchronize()
    assert (k == 7).all() and (v == 7).all()
    L.close()
