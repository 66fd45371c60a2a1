"""A decode stack's step captured into a graph and replayed by the caller, on streams that the
stack does not know, between prepares that fork, copy and move pages."""
import ctypes

import numpy as np
import pytest

import si_amd
from oracle.oracle_py import make_shape as or_shape
from tests.gpu_helpers import dev, device_view, empty, make_layer

pytestmark = pytest.mark.gpu
NL, SEQS, PS, NPAGES = 2, 4, 16, 40


class Stack:
    def __init__(self, oracle, fmt, max_ctx):
        import torch
        self.torch, self.H = torch, si_amd.host_lib()
        sd = si_amd.SHAPES["0.5b"]
        s, os_ = si_amd.make_shape(**sd), or_shape(**sd)
        self.lays = [make_layer(oracle, os_, 60 + l) for l in range(NL)]
        self.keep = [{k: np.ascontiguousarray(v) for k, v in t.items() if v is not None}
                     for t in self.lays]
        hosts = (si_amd.LayerHost * NL)(*[
            si_amd.LayerHost(**{k: v.ctypes.data for k, v in kk.items()}) for kk in self.keep])
        self.s, self.fmt, self.max_ctx, self.mp = s, fmt, max_ctx, -(-max_ctx // PS)
        self.st = self.H.si_stack_create_kv(ctypes.byref(s), ctypes.cast(hosts, ctypes.c_void_p),
                                            NL, SEQS, max_ctx, NPAGES, PS, fmt)
        self.pg = self.H.si_stack_pages(self.st)
        kvd = s.kvheads * s.hdim
        self.page = PS * kvd * 9 // 16 if fmt else PS * kvd * 2
        self.pools = [[device_view(f(self.st, l), NPAGES * self.page, torch.uint8)
                       for f in (self.H.si_stack_k_pool, self.H.si_stack_v_pool)]
                      for l in range(NL)]
        for pair in self.pools:
            for t in pair:
                t.zero_()
        torch.cuda.synchronize()

    def prepare(self, seqs):
        ids = (ctypes.c_int * len(seqs))(*seqs)
        assert self.H.si_stack_prepare(self.st, ids, len(seqs)) == 0

    def decode(self, x, out, stream=None):
        self.H.si_stack_decode(self.st, si_amd.ptr(x), si_amd.ptr(out), si_amd.SI_LAYER_FULL,
                               si_amd.stream_handle(stream))

    def rows(self, seq):
        """The bytes of a sequence's whole pages in every pool."""
        t = np.ctypeslib.as_array(self.H.si_kv_page_table(self.pg), shape=(SEQS * self.mp,))
        n = self.H.si_kv_seq_len(self.pg, seq) // PS
        ids = self.torch.from_numpy(t.reshape(SEQS, self.mp)[seq, :n].astype(np.int64)).cuda()
        return [p.view(NPAGES, self.page)[ids].clone() for pair in self.pools for p in pair]

    def close(self):
        self.H.si_stack_destroy(self.st)


@pytest.mark.parametrize("fmt", [si_amd.SI_KV_F16, si_amd.SI_KV_Q4])
def test_prepare_waits_for_replays(oracle, fmt):
    """The call returns after the replay that was running, whose pages it copies."""
    import torch
    S = Stack(oracle, fmt, 96)
    rng = np.random.default_rng(1)
    x, out = dev(rng.standard_normal((2, S.s.hidden)).astype(np.float32)), empty(
        (2, S.s.hidden), torch.float32)
    a, b = S.H.si_kv_seq_add(S.pg), S.H.si_kv_seq_add(S.pg)
    for _ in range(5):
        S.prepare([a, b])
        S.decode(x, out)
    S.prepare([a, b])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        S.decode(x, out)
    side = torch.cuda.Stream()
    ended = torch.cuda.Event()

    def replay():
        with torch.cuda.stream(side):
            torch.cuda._sleep(20000000)
            g.replay()
            ended.record()

    replay()
    c = S.H.si_stack_fork(S.st, a)  # its page is copied by the next prepare
    S.prepare([b, c])
    assert ended.query()
    replay()
    S.H.si_kv_seq_free(S.pg, a)
    S.H.si_stack_compact(S.st)
    assert ended.query()
    S.prepare([b, c])
    replay()
    S.prepare([b, c])
    assert ended.query()
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    S.close()


def test_replays_of_growing_contexts(oracle):
    """A 4-bit step captured once, replayed as its sequences grow past every context that it was
    captured with: the bits of its layers called for the stack's longest contexts."""
    import torch
    S = Stack(oracle, si_amd.SI_KV_Q4, 200)
    layers = [si_amd.Layer(S.s, lay, SEQS, S.max_ctx) for lay in S.lays]
    mem = [[t.clone() for t in pair] for pair in S.pools]
    rng = np.random.default_rng(2)
    seqs = [S.H.si_kv_seq_add(S.pg) for _ in range(3)]
    x, out = empty((3, S.s.hidden), torch.float32), empty((3, S.s.hidden), torch.float32)
    graph = None
    for step in range(40):
        if step == 20:
            S.H.si_kv_seq_truncate(S.pg, seqs[1], 4)
        S.prepare(seqs)
        x.copy_(dev(rng.standard_normal((3, S.s.hidden)).astype(np.float32)))
        torch.cuda.synchronize()
        if graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                S.decode(x, out)
        graph.replay()
        table = np.ctypeslib.as_array(S.H.si_kv_page_table(S.pg), shape=(SEQS * S.mp,)).reshape(
            SEQS, S.mp)
        tab = dev(table[seqs].copy())
        ctx = dev(np.array([S.H.si_kv_seq_len(S.pg, i) for i in seqs], np.int32))
        cur = x
        for L, (k, v) in zip(layers, mem):
            o = empty((3, S.s.hidden), torch.float32)
            L.decode_kv4(cur, 3, k, v, NPAGES, PS, tab, S.mp, ctx, S.max_ctx, o, capture=False)
            cur = o
        torch.cuda.synchronize()
        assert torch.equal(out, cur), step
        for a, b in zip(S.pools, mem):
            assert all(torch.equal(s, t) for s, t in zip(a, b)), step
    S.close()
    for L in layers:
        L.close()
