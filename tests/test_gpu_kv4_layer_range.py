"""si_layer_decode_kv4 with device contexts outside 1..max_ctx: past max_ctx they are max_ctx, as
in si_layer_decode_paged, whatever an earlier call left in the layer's buffers; below 1 the
sequence attends to nothing and its pages stay."""
import numpy as np
import pytest

import si_amd
from oracle.oracle_py import make_shape as or_shape
from tests import kv4_ref as ref
from tests.gpu_helpers import dev, empty, make_layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nseq,far", [(1, 101), (3, 101), (3, 4000), (5, 2 ** 31 - 1)])
def test_contexts_past_max_ctx(oracle, nseq, far):
    import torch
    sd = si_amd.SHAPES["0.5b"]
    s = si_amd.make_shape(**sd)
    rng, ps, max_ctx, mp = np.random.default_rng(nseq), 16, 100, 8
    L = si_amd.Layer(s, make_layer(oracle, or_shape(**sd), 21), nseq, 128)
    pools0 = [dev(ref.pack(rng.standard_normal((nseq * mp * ps, s.kvheads, s.hdim)).astype(
        np.float32), s.kvheads, s.hdim, ps, k)) for k in (True, False)]
    table = dev(rng.permutation(nseq * mp).reshape(nseq, mp).astype(np.int32))
    x, other = (dev(rng.standard_normal((nseq, s.hidden)).astype(np.float32)) for _ in "ab")

    def call(x, ctx):
        pools, out = [t.clone() for t in pools0], empty((nseq, s.hidden), torch.float32)
        L.decode_kv4(x, nseq, *pools, nseq * mp, ps, table, mp, dev(ctx), max_ctx, out,
                     capture=False)
        torch.cuda.synchronize()
        return out, pools

    inside = np.full(nseq, 40, np.int32)
    inside[-1] = max_ctx
    past = inside.copy()
    past[-1] = far
    want, held = call(x, inside)
    call(other, np.full(nseq, 17, np.int32))  # other rows in the layer's buffers
    got, now = call(x, past)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(now, held))
    # and a sequence without positions: its pages as they were, the others' rows the same, its own
    # whatever the buffers held
    if nseq > 1:
        none = inside.copy()
        none[0] = 0
        got, now = call(x, none)
        assert torch.equal(got[1:], want[1:]) and torch.isfinite(got).all()
        call(other, np.full(nseq, 17, np.int32))
        none[0] = -7
        assert torch.equal(call(x, none)[0], got)
        page = now[0].numel() // (nseq * mp)
        own = table[0].long()
        for a, b in zip(now, pools0):
            assert torch.equal(a.view(-1, page)[own], b.view(-1, page)[own])
    L.close()
