"""The calls of a ragged step refuse what they cannot run, before anything is launched (no GPU
needed: the pointers are never followed)."""
import ctypes

import pytest

import si_amd

S = ctypes.byref(si_amd.make_shape(**si_amd.SHAPES["7b"]))
BAD_HEADS = ctypes.byref(si_amd.make_shape(896, 14, 3, 64))
BAD_DIM = ctypes.byref(si_amd.make_shape(896, 14, 2, 48))
A = 1 << 12


def tables(nseq=2, have=A, add=A, max_rows=8, window=64, sinks=4, page=16, npages=8, max_pages=4,
           pages=A, ring=A, free=A, free_out=A, held=A, held_out=A, start=A, ctx=A, seq=A, pos=A,
           slot=A, taken=A, status=A):
    return si_amd.lib().si_kv_step(nseq, have, add, max_rows, window, sinks, page, npages,
                                   max_pages, pages, ring, free, free_out, held, held_out, start,
                                   ctx, seq, pos, slot, taken, status, None)


def append(shape=S, qkv=A, ld=4608, max_rows=8, max_pos=64, pos=A, slot=A, rc=A, rs=A, q=A, k=A,
           v=A, pool_rows=128):
    return si_amd.lib().si_rope_kv_append_rows(shape, qkv, ld, max_rows, max_pos, pos, slot, rc,
                                               rs, q, k, v, pool_rows, None)


def attention(shape=S, q=A, nseq=2, max_rows=8, max_new=4, max_ctx=64, window=64, sinks=4,
              start=A, ctx=A, k=A, v=A, npages=8, page=16, pages=A, max_pages=4, out=A, qs=None,
              d=None, ws=1 << 16, ws_bytes=1 << 40):
    return si_amd.lib().si_attention_rows(shape, q, nseq, max_rows, max_new, max_ctx, window,
                                          sinks, start, ctx, k, v, npages, page, pages, max_pages,
                                          out, qs, d, None, ws, ws_bytes, None)


PAGE_CASES = [(dict(page=0), b"power of two"), (dict(page=24), b"power of two"),
              (dict(page=1 << 21), b"power of two"), (dict(npages=0), b">= 1"),
              (dict(max_pages=0), b">= 1"), (dict(max_pages=1 << 20, page=2048), b"a sequence")]
STEP_CASES = [(dict(nseq=-1), b"nseq"), (dict(nseq=1 << 16), b"nseq"),
              (dict(max_rows=-1), b"max_rows"), (dict(max_rows=1 << 24), b"max_rows"),
              (dict(window=0), b"window"), (dict(window=-5), b"window"), (dict(sinks=-1), b"sinks")]
HEAD_CASES = [(dict(shape=None), b"shape is NULL"), (dict(shape=BAD_HEADS), b"unsupported heads"),
              (dict(shape=BAD_DIM), b"unsupported heads")]


def refused(rc, why):
    assert rc == si_amd.SI_ERR_ARG and why in si_amd.lib().si_last_error(), \
        si_amd.lib().si_last_error()


@pytest.mark.parametrize("bad,why", PAGE_CASES + STEP_CASES + [
    (dict(**{k: None}), b"NULL") for k in (
        "have", "add", "pages", "ring", "free", "free_out", "held", "held_out", "start", "ctx",
        "seq", "pos", "slot", "taken", "status")])
def test_tables_refuse(bad, why):
    refused(tables(**bad), why)


@pytest.mark.parametrize("bad", [dict(ctx=16 * A), dict(start=16 * A), dict(held_out=17 * A),
                                 dict(taken=17 * A), dict(seq=16 * A), dict(pos=17 * A),
                                 dict(start=18 * A, taken=18 * A), dict(ctx=18 * A, taken=18 * A)])
def test_tables_refuse_overlaps(bad):
    apart = dict(have=16 * A, add=17 * A, ctx=2 * A, start=3 * A, taken=4 * A)
    refused(tables(**dict(apart, **bad)), b"of their own" if 18 * A in bad.values() else b"outputs")


@pytest.mark.parametrize("bad,why", HEAD_CASES + [
    (dict(max_rows=-1), b"max_rows"), (dict(max_rows=1 << 24), b"max_rows"),
    (dict(max_pos=0), b"max_pos"), (dict(ld=4607), b"ldqkv"), (dict(pool_rows=0), b"pool rows"),
    (dict(pool_rows=1 << 60), b"pool rows")] + [
    (dict(**{k: None}), b"NULL") for k in ("qkv", "pos", "slot", "rc", "rs", "q", "k", "v")] + [
    (dict(**{k: A + 8}), b"16-byte aligned") for k in ("rc", "rs", "q", "k", "v")])
def test_append_refuses(bad, why):
    refused(append(**bad), why)


@pytest.mark.parametrize("bad,why", HEAD_CASES + PAGE_CASES + STEP_CASES + [
    (dict(max_new=0), b"max_new"), (dict(max_ctx=0), b"max_ctx"), (dict(max_ctx=65), b"max_ctx"),
    (dict(npages=1 << 30, page=1 << 4), b"too large"), (dict(qs=A), b"qs without d"),
    (dict(qs=A + 2, d=A), b"4-byte"), (dict(ws=(1 << 16) + 128), b"256-byte")] + [
    (dict(**{k: None}), b"NULL") for k in ("q", "start", "ctx", "k", "v", "pages", "out")] + [
    (dict(**{k: A + 8}), b"16-byte aligned") for k in ("q", "k", "v", "out")])
def test_attention_refuses(bad, why):
    refused(attention(**bad), why)


def test_attention_workspace():
    need = si_amd.lib().si_attention_rows_workspace
    for bad in ((None, 2, 8, 4, 64, 64, 4), (BAD_DIM, 2, 8, 4, 64, 64, 4), (S, -1, 8, 4, 64, 64, 4),
                (S, 2, 8, 0, 64, 64, 4), (S, 2, 8, 4, 0, 64, 4), (S, 2, 8, 4, 64, 0, 4)):
        assert need(*bad) == 0
    # rows over a long range are split, and their parts meet in the workspace
    big = need(S, 1, 1, 1, 65536, 2 ** 31 - 1, 0)
    if big:
        refused(attention(nseq=1, max_rows=1, max_new=1, max_ctx=65536, window=2 ** 31 - 1,
                          sinks=0, page=1024, max_pages=64, npages=64, ws_bytes=big - 1),
                b"workspace too small")
        refused(attention(nseq=1, max_rows=1, max_new=1, max_ctx=65536, window=2 ** 31 - 1,
                          sinks=0, page=1024, max_pages=64, npages=64, ws=None), b"workspace")


def test_nothing_to_do():
    """No rows or no sequences: success, and nothing is launched."""
    assert append(max_rows=0, qkv=None, pos=None, slot=None) == 0
    assert attention(max_rows=0, q=None, out=None) == 0
    assert attention(nseq=0, start=None, ctx=None, pages=None) == 0


def test_attention_workspace_of_idle_sequences():
    """Sequences without rows need no room: 40 rows of 7 heads a group are 8 whole tiles of 32, and
    at most one more for each of 40 sequences, in 7 parts of 32 x 130 numbers (256 workgroups of
    4 groups x 9 tiles)."""
    need = si_amd.lib().si_attention_rows_workspace
    most = (8 + 40) * 4 * 7 * 32 * 130 * 4
    assert need(S, 65535, 40, 40, 8192, 4096, 4) == need(S, 40, 40, 40, 8192, 4096, 4) <= most


def test_attention_workspace_of_nothing():
    """No rows or no sequences need no room."""
    need = si_amd.lib().si_attention_rows_workspace
    for nseq, max_rows, max_new in ((0, 8, 4), (0, 8, 100), (2, 0, 4), (2, 0, 100), (0, 0, 1)):
        assert need(S, nseq, max_rows, max_new, 65536, 65536, 4) == 0
