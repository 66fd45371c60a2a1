"""The 4-bit cache's entry points and the page copies refuse what they cannot run,
before anything is launched (no GPU needed: the pointers are never followed)."""
import ctypes

import numpy as np
import pytest

import si_amd

S = ctypes.byref(si_amd.make_shape(**si_amd.SHAPES["7b"]))
A, ODD = 1 << 12, (1 << 12) + 8
OK_CACHE = dict(k=A, v=A, npages=8, page=16, pages=A, max_pages=4)  # 64 positions


def _cache(c):
    return c["k"], c["v"], c["npages"], c["page"], c["pages"], c["max_pages"]


def append(shape=S, qkv=A, ld=4608, ntok=2, pos0=0, step=0, max_pos=64, ctx=A, rc=A, q=A, **c):
    return si_amd.lib().si_rope_kv4_append(shape, qkv, ld, ntok, pos0, step, max_pos, ctx, rc, rc,
                                           q, *_cache(dict(OK_CACHE, **c)), None)


def write(shape=S, kin=A, vin=A, ntok=2, pos0=0, step=0, ctx=A, **c):
    return si_amd.lib().si_kv4_write(shape, kin, vin, ntok, pos0, step, ctx,
                                     *_cache(dict(OK_CACHE, **c)), None)


def read(shape=S, kout=A, vout=A, ntok=2, pos0=0, step=0, ctx=A, **c):
    return si_amd.lib().si_kv4_read(shape, *_cache(dict(OK_CACHE, **c)), ntok, pos0, step, ctx,
                                    kout, vout, None)


def attention(shape=S, q=A, nq=2, ctx=A, ctx0=0, step=0, max_ctx=64, out=A, qs=None, d=None,
              ws=1 << 16, ws_bytes=1 << 40, **c):
    return si_amd.lib().si_attention_kv4(shape, q, nq, *_cache(dict(OK_CACHE, **c)), ctx, ctx0,
                                         step, max_ctx, out, qs, d, None, ws, ws_bytes, None)


BAD_HEADS = ctypes.byref(si_amd.make_shape(896, 14, 3, 64))
BAD_DIM = ctypes.byref(si_amd.make_shape(896, 14, 2, 48))
CACHE_CASES = [
    (dict(shape=None), b"shape is NULL"), (dict(shape=BAD_HEADS), b"unsupported heads"),
    (dict(shape=BAD_DIM), b"unsupported heads"), (dict(k=None), b"NULL"), (dict(v=None), b"NULL"),
    (dict(pages=None), b"NULL"), (dict(k=ODD), b"16-byte aligned"),
    (dict(v=ODD), b"16-byte aligned"), (dict(page=8), b"power of two"),
    (dict(page=48), b"power of two"), (dict(page=1 << 17), b"power of two"),
    (dict(npages=0), b">= 1"), (dict(max_pages=0), b">= 1"),
    (dict(max_pages=1 << 20, page=1 << 16), b"a sequence"),
]
ROW_CASES = [
    (dict(ntok=-1), b"bad ntok"), (dict(pos0=-1), b"bad ntok"), (dict(step=2), b"neither"),
    (dict(step=1), b"ctx_dev goes with"), (dict(ctx=None, pos0=64), b"exceed 64"),
    (dict(ctx=None, step=1, pos0=63), b"exceed 64"),
    (dict(ctx=None, step=1, ntok=2 ** 31 - 1, pos0=2 ** 31 - 1), b"exceed"),
    (dict(ntok=1 << 24), b"2^24 - 1 rows"),
]


@pytest.mark.parametrize("call", [append, write, read, attention])
@pytest.mark.parametrize("args,msg", CACHE_CASES)
def test_cache_arguments(call, args, msg):
    assert call(**args) == si_amd.SI_ERR_ARG
    assert msg in si_amd.lib().si_last_error()


@pytest.mark.parametrize("call", [append, write, read])
@pytest.mark.parametrize("args,msg", ROW_CASES)
def test_row_arguments(call, args, msg):
    assert call(**args) == si_amd.SI_ERR_ARG
    assert msg in si_amd.lib().si_last_error()


@pytest.mark.parametrize("args,msg", [
    (dict(ld=4607), b"ldqkv"), (dict(qkv=None), b"NULL"), (dict(rc=None), b"NULL"),
    (dict(q=None), b"NULL"), (dict(max_pos=0), b"max_pos"),
    (dict(max_pos=32, ctx=None, pos0=32), b"exceed 32")])
def test_append_arguments(args, msg):
    assert append(**args) == si_amd.SI_ERR_ARG
    assert msg in si_amd.lib().si_last_error()


@pytest.mark.parametrize("call,a,b", [(write, "kin", "vin"), (read, "kout", "vout")])
def test_row_buffers(call, a, b):
    for name in (a, b):
        assert call(**{name: None}) == si_amd.SI_ERR_ARG
        assert b"NULL" in si_amd.lib().si_last_error()
        assert call(**{name: ODD}) == si_amd.SI_ERR_ARG
        assert b"16-byte aligned" in si_amd.lib().si_last_error()


@pytest.mark.parametrize("args,msg", [
    (dict(nq=-1), b"bad nq"), (dict(nq=65536), b"bad nq"), (dict(max_ctx=0), b"max_ctx"),
    (dict(max_ctx=65), b"do not cover"), (dict(step=-1), b"neither"), (dict(step=2), b"neither"),
    (dict(step=1), b"ctx_dev goes with"), (dict(ctx=None), b">= 1"),
    (dict(ctx=None, ctx0=65), b"exceeds max_ctx"), (dict(ctx=None, ctx0=64, step=1), b"exceeds"),
    (dict(q=None), b"NULL"), (dict(out=None), b"NULL"), (dict(qs=A), b"qs without d")])
def test_attention_arguments(args, msg):
    assert attention(**args) == si_amd.SI_ERR_ARG
    assert msg in si_amd.lib().si_last_error()


def test_attention_workspace():
    L = si_amd.lib()
    for nq, step, max_ctx in ((0, 0, 64), (1, 0, 0), (1, 2, 64), (1, -1, 64)):
        assert L.si_attention_kv4_workspace(S, nq, step, max_ctx) == 0
    assert L.si_attention_kv4_workspace(BAD_HEADS, 1, 0, 64) == 0
    need = L.si_attention_kv4_workspace(S, 2, 1, 64)
    if need:
        for bad in (dict(ws_bytes=need - 1), dict(ws=None), dict(ws=(1 << 16) + 16)):
            assert attention(ctx=None, ctx0=1, step=1, **bad) == si_amd.SI_ERR_ARG
            assert b"workspace" in L.si_last_error()


def test_workspace_of_long_prompts():
    """A prompt of more than 9000 (query, head) rows takes fp16 rows of max_ctx positions, but
    not past 2^26 of them; the largest contexts do not wrap."""
    L = si_amd.lib()
    rows = lambda n: L.si_attention_kv4_workspace(S, 400, 1, n)
    assert rows(1 << 16) == (1 << 16) * 4 * 128 * 4 and rows(1 << 26) == (1 << 26) * 4 * 128 * 4
    assert rows((1 << 26) + 1) < 1 << 28
    for nq, step in ((1, 0), (64, 0), (400, 1)):
        a, b = (L.si_attention_kv4_workspace(S, nq, step, n) for n in (1 << 30, 2 ** 31 - 1))
        assert a == b > 0


def test_no_rows_is_no_work():
    assert append(ntok=0, qkv=None, rc=None, q=None) == si_amd.SI_OK
    assert write(ntok=0, kin=None, vin=None) == si_amd.SI_OK
    assert read(ntok=0, kout=None, vout=None) == si_amd.SI_OK
    assert attention(nq=0, q=None, out=None) == si_amd.SI_OK


def test_page_bytes():
    f = si_amd.lib().si_kv4_page_bytes
    assert f(S, 64) == 4 * 64 * 128 * 9 // 16
    assert f(ctypes.byref(si_amd.make_shape(**si_amd.SHAPES["0.5b"])), 16) == 2 * 16 * 64 * 9 // 16
    assert f(BAD_HEADS, 64) == 0 and f(None, 64) == 0 and f(S, 24) == 0 and f(S, 8) == 0


def copy(pools, page_bytes, npages, src, dst, n=None):
    p = (ctypes.c_void_p * max(len(pools), 1))(*pools)
    s, d = (np.asarray(x, np.int32) for x in (src, dst))
    return si_amd.lib().si_kv_copy_pages(p, len(pools), page_bytes, npages, si_amd.ptr(s),
                                         si_amd.ptr(d), len(s) if n is None else n, None)


def test_copy_arguments():
    L, far = si_amd.lib(), 1 << 30
    for args, msg in (
            (([A], 64, 0, [0], [1]), b"bad sizes"), (([A], 0, 4, [0], [1]), b"bad sizes"),
            (([A], 64, 4, [0], [1], -1), b"bad sizes"),
            (([A], 1 << 39, 4, [0], [1]), b"pages of"), (([A, None], 64, 4, [0], [1]), b"NULL"),
            (([A], 64, 4, [0], [4]), b"outside 0..3"), (([A], 64, 4, [-1], [1]), b"outside"),
            (([A], 64, 4, [4], [1]), b"outside"), (([A], 64, 4, [0], [-1]), b"outside"),
            (([A], 64, 4, [0, 1], [2, 2]), b"page 2 is written twice"),
            (([A], 64, 4, [0, 1], [1, 2]), b"page 1 is read and written"),
            (([A], 64, 4, [1], [1]), b"page 1 is read and written"),
            (([A, A], 64, 4, [0], [1]), b"overlap"),
            (([far, A, A + 255], 64, 4, [0], [1]), b"overlap")):
        assert copy(*args) == si_amd.SI_ERR_ARG, args
        assert msg in L.si_last_error(), (args, L.si_last_error())
    assert L.si_kv_copy_pages(None, 1, 64, 4, None, None, 0, None) == si_amd.SI_ERR_ARG
    assert L.si_kv_copy_pages(ctypes.byref(ctypes.c_void_p(A)), 1, 64, 4, None, None, 1,
                              None) == si_amd.SI_ERR_ARG
    assert copy([A, A + 256], 64, 4, [], []) == si_amd.SI_OK  # no moves
    assert copy([], 64, 4, [0], [1]) == si_amd.SI_OK  # no pools
