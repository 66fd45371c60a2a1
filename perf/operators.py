"""The operators of a K/V cache held in 4 bits, and of its pages, case by case.

A server whose memory is the cache keeps K and V rows in 4 bits: blocks of 32 values of a
row share a scale, and a page of such rows takes 9/32 of an fp16 page.  Its operators are
  append     RoPE of a step's q|k|v rows, K and V quantized into the pages (one token for each
             of a batch of sequences, or a prompt of one), the rotated q handed on
  store      fp16 cache rows into the pages, as after a prompt that ran over an fp16 cache
  attention  GQA attention over the pages, a query per sequence, or a prompt's (causal)
  copy       pages copied to others in every pool of a model: forks, and compaction
append and store return the rows as the cache holds them (read back through the library).

The block: m its value of largest magnitude (the negative one of a pair, a NaN taken as 0),
h = -m / 128 limited to +-508, rounded to 7 significant bits and to fp16; a value x becomes
n = floor(x / (16 h) + 8.5), exactly, limited to 0..15 (8 where h is 0) and stands for 16 h (n - 8),
which fp16 holds exactly.  A page holds for each KV head the nibbles of its positions and
then their scales:
  K nibbles  [pos / 8][pos / 4 % 2][dim / 8 % 4][pos % 4][dim / 32][dim % 8]
  V nibbles  [pos / 8][16 dims' groups in fours, then a pair][dim % 16][group][pos % 8]
  scales     [pos / 8][dim / 32][pos % 4][pos / 4 % 2] fp16
Everything is made from the seed, on the GPU.
"""
import ctypes
import math

import torch

own = False
DEV = "cuda"
BLK = 32


def listed():
    small, big, mid = (dict(qheads=q, kvheads=k, hdim=d)
                       for q, k, d in ((14, 2, 64), (28, 4, 128), (12, 2, 128)))
    return [
        # one user's next token on a small model: latency
        dict(name="append_one", op="append", **small, rows=1, low=777, high=777, prompt=False,
             page=16),
        # a busy server's step: a token for each of 64 users at different points
        dict(name="append_batch", op="append", **big, rows=64, low=40, high=4096, prompt=False,
             page=64),
        # the next piece of a long prompt, starting and ending inside a page
        dict(name="append_prompt", op="append", **big, rows=1999, low=333, high=333, prompt=True,
             page=64),
        # the last piece of a prompt that ran over an fp16 cache
        dict(name="store_piece", op="store", **small, rows=77, first=1003, page=16),
        # a whole prompt's fp16 cache
        dict(name="store_prompt", op="store", **mid, rows=5000, first=0, page=32),
        # one user's next token over a short context: latency
        dict(name="attention_one", op="attention", **small, rows=1, low=1024, high=1024, page=16),
        # a server's users at different points of their chats
        dict(name="attention_ragged", op="attention", **big, rows=48, low=200, high=4096,
             page=64),
        # every user at the longest context
        dict(name="attention_full", op="attention", **big, rows=64, low=4096, high=4096, page=64),
        # two users with documents: few rows, a very long axis
        dict(name="attention_long", op="attention", **mid, rows=2, low=60000, high=131072,
             page=256),
        # the next piece of a prompt over what the cache holds
        dict(name="attention_prompt", op="prompt", **big, rows=333, first=1500, page=64),
        # a fork of a sequence before its next token: its last pages, in all 28 layers' pools
        dict(name="copy_fork", op="copy", pools=56, words=4608, pages=200, moved=3),
        # fp16 pools compacted before half of them is given back
        dict(name="copy_compact", op="copy", pools=16, words=16384, pages=1200, moved=500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((14, 2, 64), (28, 4, 128), (12, 2, 128), (32, 2, 64), (24, 8, 96), (8, 8, 32),
         (16, 1, 128))


def draw(rng):
    op = rng.choice(["append", "append", "store", "attention", "attention", "attention",
                     "prompt", "copy"])
    if op == "copy":
        words = 64 * rng.choice([16, 20, 32, 72, 128, 144, 256])
        pools, moved = _log(rng, 1, 64), _log(rng, 1, 500)
        moved = max(1, min(moved, 131072000 // (words * pools)))
        return dict(op=op, pools=pools, words=words, pages=2 * moved + rng.randint(1, 100),
                    moved=moved)
    q, k, d = rng.choice(HEADS)
    c = dict(op=op, qheads=q, kvheads=k, hdim=d, page=rng.choice([16, 32, 64, 128]))
    if op == "append":
        prompt = rng.random() < 0.5
        low = rng.randint(1, 3000)
        return dict(c, rows=_log(rng, 1, 1900 if prompt else 200), low=low,
                    high=low if prompt else low + rng.randint(0, 3000), prompt=prompt)
    if op == "store":
        return dict(c, rows=_log(rng, 1, 2500), first=rng.choice([0, rng.randint(1, 2000)]))
    if op == "prompt":
        return dict(c, rows=_log(rng, 2, 333), first=rng.choice([0, _log(rng, 1, 1500)]))
    rows = _log(rng, 1, 64)
    # positions times KV width stay below the largest listed case's
    high = _log(rng, 16, min(100000, 64 * 4096 * 512 // (rows * k * d)))
    return dict(c, rows=rows, low=rng.randint(0, high), high=high)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _State:
    pass


class _Inputs:
    """Seeded tensors on the GPU, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 29)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV)

    def rows(self, n, width):
        """n rows of width values whose channels differ in size, some by far, as a
        projection's do."""
        size = torch.exp(0.5 * self.normal(width)) * torch.where(
            torch.rand(width, generator=self.g, device=DEV) < 0.02, 12.0, 1.0)
        return self.normal(n, width) * size

    def contexts(self, n, low, high):
        c = torch.randint(low, high + 1, (n,), generator=self.g, device=DEV, dtype=torch.int32)
        c[n // 2] = high
        return c

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=DEV).to(torch.int32)


def _page_bytes(c):
    """Bytes of one KV head's part of a page."""
    return c["page"] * c["hdim"] * 9 // 16


def _quantize(x):
    """(nibbles 0..15, fp16 scales) of the 32-value blocks of x [..., hdim]."""
    b = torch.nan_to_num(x.float(), nan=0.0, posinf=math.inf, neginf=-math.inf)
    b = b.view(*x.shape[:-1], -1, BLK)
    top, bottom = b.amax(-1), b.amin(-1)
    m = torch.where(-bottom >= top, bottom, top)
    t = (m * -0.0078125).clamp(-508.0, 508.0)
    u = t.view(torch.int32)
    u = (u + 0xffff + ((u >> 17) & 1)) & -0x20000  # to 7 significant bits, ties to even
    h = u.view(torch.float32).half()
    d = h.double()[..., None] * 16  # 64 bits: a quotient next to a border keeps its side
    n = torch.where(d == 0, 8.0, (b.double() / d + 8.5).floor().clamp(0, 15))
    return n.to(torch.uint8).view(x.shape), h


def _value(n, h):
    """fp32 values of nibbles n [..., hdim] and scales h [..., hdim / 32]."""
    b = n.view(*h.shape, BLK).float() - 8
    return (b * (h.float() * 16)[..., None]).view(n.shape)


def _bytes(nib):
    """Nibbles [..., 8] as 4 bytes, the first in the low bits."""
    return nib[..., 0::2] | nib[..., 1::2] << 4


def _nibbles(b):
    """Bytes [..., 4] as 8 nibbles."""
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _lay_out(n, h, is_k):
    """Pages [P][kvheads][page * hdim * 9 / 16] of nibbles n [P][kvheads][page][hdim] and
    scales h [P][kvheads][page][hdim / 32]."""
    P, kv, ps, D = n.shape
    if is_k:
        w = n.view(P, kv, ps // 8, 2, 4, D // 32, 4, 8).permute(0, 1, 2, 3, 6, 4, 5, 7)
        nib = _bytes(w).reshape(P, kv, ps // 8, 4 * D)
    else:
        w = n.view(P, kv, ps // 8, 8, D // 16, 16)
        full = D // 64 * 4
        parts = []
        if full:
            a = w[..., :full, :].reshape(P, kv, ps // 8, 8, full // 4, 4, 16)
            parts.append(_bytes(a.permute(0, 1, 2, 4, 6, 5, 3)).reshape(P, kv, ps // 8, -1))
        if full < D // 16:
            a = w[..., full:, :].permute(0, 1, 2, 5, 4, 3)
            parts.append(_bytes(a).reshape(P, kv, ps // 8, -1))
        nib = torch.cat(parts, -1)
    s = h.view(P, kv, ps // 8, 2, 4, D // 32).permute(0, 1, 2, 5, 4, 3).contiguous()
    return torch.cat([nib.reshape(P, kv, -1), s.view(torch.uint8).reshape(P, kv, -1)],
                     -1).contiguous()


def _values(pages, ps, D, is_k):
    """fp32 [..., kvheads][ps][D] of pages [..., kvheads][bytes]."""
    lead = pages.shape[:-1]
    nib, s = pages.split([ps * D // 2, ps * D // 16], -1)
    h = s.contiguous().view(torch.float16).view(-1, ps // 8, D // 32, 4, 2)
    h = h.permute(0, 1, 4, 3, 2).reshape(*lead, ps, D // 32)
    nib = nib.reshape(-1, ps // 8, 4 * D)
    if is_k:
        n = _nibbles(nib.reshape(-1, ps // 8, 2, 4, 4, D // 32, 4))
        n = n.permute(0, 1, 2, 4, 5, 3, 6)
    else:
        full = D // 64 * 4
        a, b = nib.split([64 * full, 4 * D - 64 * full], -1)
        parts = []
        if full:
            x = _nibbles(a.reshape(-1, ps // 8, full // 4, 16, 4, 4))
            parts.append(x.permute(0, 1, 5, 2, 4, 3).reshape(-1, ps // 8, 8, full * 16))
        if full < D // 16:
            x = _nibbles(b.reshape(-1, ps // 8, 16, 2, 4))
            parts.append(x.permute(0, 1, 4, 3, 2).reshape(-1, ps // 8, 8, 32))
        n = torch.cat(parts, -1)
    return _value(n.reshape(*lead, ps, D), h)


def _pool(r, c, n):
    """n pages of rows as a cache holds them (K of moderate size, so that scores spread)."""
    ps, kv, D = c["page"], c["kvheads"], c["hdim"]
    two = []
    for is_k in (True, False):
        x = r.rows(n * ps, kv * D) * (0.5 if is_k else 1.0)
        x = x.view(n, ps, kv, D).transpose(1, 2).contiguous()
        two.append(_lay_out(*_quantize(x), is_k))
    return two


def _table(npos, D):
    i = torch.arange(D // 2, device=DEV, dtype=torch.float64)
    a = torch.arange(npos, device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-2 * i / D)
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    r, s, c = _Inputs(seed), _State(), case
    s.case, op = c, c["op"]
    if op == "copy":
        s.pools = torch.randint(-2 ** 31, 2 ** 31, (c["pools"], c["pages"], c["words"]),
                                generator=r.g, device=DEV, dtype=torch.int32)
        ids = r.order(c["pages"])
        s.src, s.dst = ids[:c["moved"]].long(), ids[c["moved"]:2 * c["moved"]].long()
        # the program's own lists: pool addresses and page ids, on the host
        ints, addr = ctypes.c_int * c["moved"], ctypes.c_void_p * c["pools"]
        s.src_host, s.dst_host = ints(*s.src.tolist()), ints(*s.dst.tolist())
        s.addr = addr(*(p.data_ptr() for p in s.pools))
        return s
    q, kv, D, n, ps = c["qheads"], c["kvheads"], c["hdim"], c["rows"], c["page"]
    one = op in ("store", "prompt") or c.get("prompt")  # rows of one sequence
    if one:
        first = c["first"] if "first" in c else c["low"]
        s.first, longest, seqs = first, first + n, 1
    else:
        s.first, longest, seqs = 0, c["high"], n
    s.max_pages = (longest + ps - 1) // ps
    s.npages = seqs * s.max_pages
    s.pages = r.order(s.npages).view(seqs, s.max_pages)
    s.max_ctx = longest
    if op in ("append", "store"):
        shape = (s.npages, kv, _page_bytes(c))
        s.k, s.v = (torch.zeros(shape, dtype=torch.uint8, device=DEV) for _ in range(2))
        s.k16, s.v16 = (torch.empty(n, kv * D, dtype=torch.float16, device=DEV)
                        for _ in range(2))
    else:
        s.k, s.v = _pool(r, c, s.npages)
    s.ctx = None if one else r.contexts(n, c["low"], c["high"])
    if op == "append":
        s.qkv = r.rows(n, (q + 2 * kv) * D)
        s.cos, s.sin = _table(longest, D)
        s.pos = (torch.arange(s.first, longest, device=DEV) if one else s.ctx.long() - 1)
        s.q = torch.empty(n, q * D, device=DEV)
    elif op == "store":
        s.kc, s.vc = (r.rows(longest, kv * D).half() for _ in range(2))
    else:
        s.q = r.normal(n, q * D)
        s.out = torch.empty(n, q * D, device=DEV)
        s.last = (torch.arange(s.first + 1, longest + 1, device=DEV) if one else s.ctx.long())
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_rope(x, cos, sin, heads):
    a, b = x.view(x.shape[0], heads, 2, -1).unbind(2)
    c, s = cos[:, None], sin[:, None]
    return torch.stack([a * c - b * s, b * c + a * s], 2).view(x.shape)


def _plain_held(x, kv, D):
    """Rows [n][kvheads * hdim] as the cache holds them, in fp16."""
    return _value(*_quantize(x.reshape(-1, kv, D))).half().view(x.shape)


def _plain_attend(q, k, v, last):
    """q [n][kv][G][D], k and v [n][kv][L][D]: query i over its first last[i] positions."""
    t = torch.matmul(k, q.transpose(2, 3).contiguous()) / math.sqrt(q.shape[3])  # [n][kv][L][G]
    seen = torch.arange(k.shape[2], device=DEV)[None, :] < last[:, None]
    t = t.masked_fill(~seen[:, None, :, None], -math.inf)
    top = t.amax(2, keepdim=True).clamp(min=-1e30)
    p = torch.exp(t - top)
    total = p.sum(2)[..., None]  # [n][kv][G][1]; 0 where nothing is seen
    out = torch.matmul(p.transpose(2, 3).contiguous(), v)
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _plain_prompt(q, k, v, last, heads, kv, D):
    """Queries q [n][heads * D] of one sequence over k and v [kv][L][D]."""
    n, G = q.shape[0], heads // kv
    q = q.view(n, kv, G, D).permute(1, 2, 0, 3).reshape(kv, G * n, D)
    t = torch.matmul(q, k.transpose(1, 2).contiguous()).view(kv, G, n, -1) / math.sqrt(D)
    seen = torch.arange(k.shape[1], device=DEV)[None, :] < last[:, None]
    t = t.masked_fill(~seen, -math.inf)
    p = torch.exp(t - t.amax(3, keepdim=True))
    total = p.sum(3, keepdim=True)
    out = torch.matmul(p.view(kv, G * n, -1), v).view(kv, G, n, D) / total
    return out.permute(2, 0, 1, 3).reshape(n, heads * D)


def _plain(s):
    c, op = s.case, s.case["op"]
    if op == "copy":
        s.pools[:, s.dst] = s.pools[:, s.src]
        return dict(pools=s.pools)
    q, kv, D, n, ps = c["qheads"], c["kvheads"], c["hdim"], c["rows"], c["page"]
    if op == "append":
        cos, sin = s.cos[s.pos], s.sin[s.pos]
        a, k, v = s.qkv.split([q * D, kv * D, kv * D], 1)
        return dict(q=_plain_rope(a, cos, sin, q),
                    k=_plain_held(_plain_rope(k, cos, sin, kv), kv, D), v=_plain_held(v, kv, D))
    if op == "store":
        return dict(k=_plain_held(s.kc[s.first:], kv, D), v=_plain_held(s.vc[s.first:], kv, D))
    k, v = (_values(t[s.pages.long()], ps, D, is_k).transpose(1, 2).reshape(
        s.pages.shape[0], kv, -1, D) for t, is_k in ((s.k, True), (s.v, False)))
    if op == "prompt":
        return dict(out=_plain_prompt(s.q, k[0], v[0], s.last, q, kv, D))
    return dict(out=_plain_attend(s.q.view(n, kv, q // kv, D), k, v, s.last).view(n, q * D))


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
_kept = {}


def _library():
    if "lib" not in _kept:
        import os
        import sys
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "simple-inference_amd"))
        import si_amd
        _kept["lib"] = si_amd
    return _kept["lib"]


def _workspace(nbytes):
    """The program's one workspace, as large as its calls have needed."""
    if "ws" not in _kept or _kept["ws"].numel() < nbytes:
        _kept["ws"] = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=DEV)
    return _kept["ws"]


def _own(s):
    si, c, op = _library(), s.case, s.case["op"]
    p, call, st = si.ptr, si.call, si.stream_handle()
    if op == "copy":
        call("si_kv_copy_pages", s.addr, c["pools"], 4 * c["words"], c["pages"], s.src_host,
             s.dst_host, c["moved"], st)
        return dict(pools=s.pools)
    n, ps = c["rows"], c["page"]
    shape = ctypes.byref(si.make_shape(32, c["qheads"], c["kvheads"], c["hdim"]))
    cache = (p(s.k), p(s.v), s.npages, ps, p(s.pages), s.max_pages)
    if op in ("append", "store"):
        step = int(s.ctx is None)
        if op == "append":
            call("si_rope_kv4_append", shape, p(s.qkv), s.qkv.shape[1], n, s.first, step,
                 s.cos.shape[0], p(s.ctx), p(s.cos), p(s.sin), p(s.q), *cache, st)
        else:
            row = c["kvheads"] * c["hdim"] * 2 * s.first
            call("si_kv4_write", shape, s.kc.data_ptr() + row, s.vc.data_ptr() + row, n, s.first,
                 step, p(s.ctx), *cache, st)
        call("si_kv4_read", shape, *cache, n, s.first, step, p(s.ctx), p(s.k16), p(s.v16), st)
        held = dict(k=s.k16, v=s.v16)
        return dict(held, q=s.q) if op == "append" else held
    step = int(s.ctx is None)
    need = si.lib().si_attention_kv4_workspace(shape, n, step, s.max_ctx)
    ws = _workspace(need)
    call("si_attention_kv4", shape, p(s.q), n, *cache, p(s.ctx), s.first + 1, step, s.max_ctx,
         p(s.out), None, None, None, p(ws), need, st)
    return dict(out=s.out)


def run(s):
    return _own(s) if own else _plain(s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Every live cache row, input and output once; two operations per multiply and add of the
    two products, six per rotated pair, four per quantized value."""
    c, op = case, case["op"]
    if op == "copy":
        return dict(bytes=8.0 * c["pools"] * c["words"] * c["moved"], flops=0.0)
    q, kv, D, n = c["qheads"], c["kvheads"], c["hdim"], c["rows"]
    qd, kvd = q * D, kv * D
    held = 2 * kvd * 9 / 16  # a position's K and V in the pages
    if op == "append":  # rows in, q and pages out, pages in, fp16 rows out
        return dict(bytes=n * (4 * (qd + 2 * kvd) + 4 * D + 4 * qd + 2 * held + 4 * kvd),
                    flops=n * (3.0 * (qd + kvd) + 8.0 * kvd))
    if op == "store":
        return dict(bytes=n * (4 * kvd + 2 * held + 4 * kvd), flops=n * 8.0 * kvd)
    if op == "prompt":
        seen, rows = n * c["first"] + n * (n + 1) / 2, c["first"] + n
    else:
        seen = rows = (n - 1) * (c["low"] + c["high"]) / 2 + c["high"]
    return dict(bytes=rows * held + 8 * n * qd, flops=4.0 * seen * qd)


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _held64(x):
    """Rows as the cache holds them: every step of the block's definition in 64 bits."""
    b = x.double().reshape(x.shape[0], -1, BLK)
    at = b.abs().max(-1, keepdim=True).values
    m = torch.where((b == -at).any(-1, keepdim=True), -at, at)
    t = (-m / 128).clamp(-508, 508)
    e = torch.frexp(t).exponent.double()  # |t| in [2^(e-1), 2^e)
    step = torch.exp2(e - 7)
    h = torch.round(torch.round(t / step) * step * 2.0 ** 24) / 2.0 ** 24
    n = torch.where(h == 0, torch.full_like(b, 8.0),
                    torch.floor(b / (16 * h) + 0.5 + 8).clamp(0, 15))
    return (16 * h * (n - 8)).reshape(x.shape)


def _read64(pool, ids, n, c, is_k):
    """The first n positions of a page list as 64-bit values [kvheads][n][hdim], byte by byte."""
    ps, D = c["page"], c["hdim"]
    pos, e = torch.arange(n, device=DEV)[:, None], torch.arange(D, device=DEV)[None, :]
    i = pos % ps
    u = i // 8
    if is_k:
        at = (u * 4 * D + i // 4 % 2 * 2 * D + e // 8 % 4 * (D // 2) + i % 4 * (D // 8)
              + e // 32 * 4 + e % 8 // 2)
        odd = e % 2 + 0 * i
    else:
        g, full = e // 16, D // 64 * 4
        fours = g // 4 * 256 + e % 16 * 16 + g % 4 * 4
        pair = full * 64 + e % 16 * 8 + (g - full) * 4
        at = u * 4 * D + torch.where(g < full, fours, pair) + i % 8 // 2
        odd = i % 2 + 0 * e
    sc = ps * D // 2 + (u * (D // 32) + e // 32) * 16 + (i % 4 * 2 + i // 4 % 2) * 2
    rows = pool[ids.long()]  # [pages of the sequence][kvheads][bytes]
    kv, size = rows.shape[1], rows.shape[2]
    flat = rows.transpose(0, 1).reshape(kv, -1)
    base = pos // ps * size
    byte = flat[:, (base + at).view(-1)].view(kv, n, D).int()
    nib = torch.where(odd == 1, byte >> 4, byte & 15)
    lo, hi = (flat[:, (base + sc + k).view(-1)].view(kv, n, D).int() for k in (0, 1))
    bits = lo | hi << 8
    sign = 1 - 2 * (bits >> 15)
    ex, man = bits >> 10 & 31, (bits & 1023).double()
    h = torch.where(ex > 0, (1 + man / 1024) * torch.exp2((ex - 15).double()), man * 2.0 ** -24)
    return sign * h * 16 * (nib - 8)


def exact(case, seed):
    c, op = case, case["op"]
    s = prepare(case, seed)
    if op == "copy":
        want = s.pools.clone()
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            want[:, b] = s.pools[:, a]
        return dict(pools=want)
    q, kv, D, n = c["qheads"], c["kvheads"], c["hdim"], c["rows"]
    if op == "store":
        return dict(k=_held64(s.kc[s.first:]), v=_held64(s.vc[s.first:]))
    if op == "append":
        x = s.qkv.double().view(n, q + 2 * kv, D)
        cos, sin = s.cos.double()[s.pos][:, None], s.sin.double()[s.pos][:, None]
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        y = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
        return dict(q=y[:, :q].reshape(n, -1), k=_held64(y[:, q:q + kv].reshape(n, -1)),
                    v=_held64(x[:, q + kv:].reshape(n, -1)))
    out = torch.zeros(n, q, D, device=DEV, dtype=torch.float64)
    qq, last = s.q.double().view(n, q, D), s.last.tolist()
    G = q // kv
    k = v = None
    for i in range(1 if op == "prompt" else n):
        if last[i] == 0:
            continue
        m = s.max_ctx if op == "prompt" else last[i]
        k, v = (_read64(t, s.pages[i], m, c, is_k) for t, is_k in ((s.k, True), (s.v, False)))
        for h in range(q):
            rows = slice(None) if op == "prompt" else slice(i, i + 1)
            t = qq[rows, h] @ k[h // G].T.contiguous() / math.sqrt(D)
            if op == "prompt":
                t = t.masked_fill(torch.arange(m, device=DEV)[None] >= s.last[:, None], -math.inf)
            out[rows, h] = torch.softmax(t, 1) @ v[h // G]
    return dict(out=out.view(n, q * D))
