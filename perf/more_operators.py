"""The operators of a step whose sequences bring any number of rows each, case by case.

A server that decodes, checks drafted tokens and takes in prompts piece by piece runs them all in
one step over a paged fp16 cache.  Its attention sees a sliding window and a few first tokens
(sinks), so that old pages can be given back, and its lengths and page lists stay on the GPU:
  step       from each sequence's length and new rows: page lists (pages taken from a ring of free
             ones, those that fell out of the window put back), the rows' sequences, positions and
             pool rows
  append     RoPE of the step's q|k|v rows, K and V to their pool rows, the rotated q handed on
  attention  GQA attention of the step's rows over the pages: row p of a sequence sees position
             t <= p where t > p - window or t < sinks

A sequence's state is a pair (pages taken so far, pages given back): its list's first
ceil(sinks / page) pages stay, the next ones given back are gone.  The ring's state is a pair
(where its free ids begin, how many there are).  A sequence of length -1 has ended: all of its
pages go back.  Everything is made from the seed, on the GPU.
"""
import ctypes
import math

import torch

own = False
DEV = "cuda"


def listed():
    small, big, mid = (dict(qheads=q, kvheads=k, hdim=d)
                       for q, k, d in ((14, 2, 64), (28, 4, 128), (12, 2, 128)))
    return [
        # one user's five drafted tokens: latency
        dict(name="step_one", op="step", seqs=1, low=777, high=777, new=5, most=5, pieces=0,
             piece=0, page=16, window=4096, sinks=4),
        # a busy server's step: a token or a few drafted ones for each of 200 users
        dict(name="step_batch", op="step", seqs=200, low=40, high=9000, new=1, most=8, pieces=0,
             piece=0, page=64, window=4096, sinks=4),
        # the tables of a whole fleet: many users, and prompts taken in
        dict(name="step_fleet", op="step", seqs=4000, low=1, high=6000, new=0, most=5, pieces=40,
             piece=2000, page=16, window=1024, sinks=4),
        # drafted tokens of eight users of a small model
        dict(name="append_draft", op="append", **small, seqs=8, low=100, high=2000, new=5, most=5,
             pieces=0, piece=0, page=16),
        # single tokens among pieces of prompts
        dict(name="append_mixed", op="append", **big, seqs=64, low=40, high=6000, new=1, most=1,
             pieces=4, piece=500, page=64),
        # one user's next token in a long chat of a small model: latency
        dict(name="attention_one", op="attention", **small, seqs=1, low=5000, high=5000,
             new=1, most=1, pieces=0, piece=0, page=16, window=1024, sinks=4),
        # a few drafted tokens of each of 16 users at different points of their chats
        dict(name="attention_draft", op="attention", **big, seqs=16, low=200, high=6000,
             new=1, most=8, pieces=0, piece=0, page=64, window=4096, sinks=4),
        # every user past the window
        dict(name="attention_batch", op="attention", **big, seqs=64, low=4200, high=20000,
             new=1, most=1, pieces=0, piece=0, page=64, window=4096, sinks=4),
        # two users with documents: few rows, a wide window
        dict(name="attention_long", op="attention", **mid, seqs=2, low=60000, high=131072,
             new=1, most=1, pieces=0, piece=0, page=256, window=65536, sinks=64),
        # the next piece of a prompt over what the cache holds
        dict(name="attention_piece", op="attention", **big, seqs=1, low=1833, high=1833,
             new=333, most=333, pieces=0, piece=0, page=64, window=1024, sinks=4),
        # single tokens among pieces of prompts
        dict(name="attention_mixed", op="attention", **big, seqs=24, low=500, high=5000,
             new=1, most=1, pieces=4, piece=300, page=64, window=2048, sinks=4),
        # a whole long prompt
        dict(name="attention_prompt", op="attention", **big, seqs=1, low=8000, high=8000,
             new=8000, most=8000, pieces=0, piece=0, page=64, window=2048, sinks=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((14, 2, 64), (28, 4, 128), (12, 2, 128), (32, 2, 64), (24, 8, 96), (8, 8, 32),
         (16, 1, 128))


def draw(rng):
    op = rng.choice(["step", "append", "attention", "attention", "attention", "attention"])
    c = dict(op=op, page=rng.choice([1, 4, 16, 32, 64, 128, 256]))
    if op != "append":
        c.update(window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 4, 16, 70]))
    if op == "step":
        seqs = _log(rng, 1, 3000)
        lo = rng.randint(0, 2)
        pieces = rng.choice([0, rng.randint(0, max(0, seqs // 50))])
        low = rng.randint(1, 3000)
        return dict(c, page=rng.choice([4, 16, 32, 64, 128]), seqs=seqs, low=low,
                    high=low + rng.randint(0, 3000), new=lo, most=lo + rng.randint(0, 8),
                    pieces=pieces, piece=_log(rng, 16, 2000))
    q, k, d = rng.choice(HEADS)
    c.update(qheads=q, kvheads=k, hdim=d)
    lo = rng.randint(0, 2)
    new = dict(new=lo, most=max(1, lo + rng.randint(0, 8)))
    if op == "append":
        seqs, low = _log(rng, 1, 100), rng.randint(1, 3000)
        return dict(c, seqs=seqs, low=low, high=low + rng.randint(0, 3000), **new,
                    pieces=rng.randint(0, min(3, seqs)), piece=_log(rng, 16, 500))
    kind = rng.choice(["rows", "rows", "piece", "mixed"])
    if kind == "piece":
        n = _log(rng, 9, 2500)
        low = n + rng.choice([0, _log(rng, 1, 1500)])
        return dict(c, seqs=1, low=low, high=low, new=n, most=n, pieces=0, piece=0)
    seqs = _log(rng, 1, 64 if kind == "rows" else 16)
    low = _log(rng, 1, 8000)
    # positions times KV width stay below the largest listed case's
    high = low + _log(rng, 1, max(2, min(100000, 64 * 4096 * 512 // (seqs * k * d))))
    if kind == "rows":
        return dict(c, seqs=seqs, low=low, high=high, **new, pieces=0, piece=0)
    return dict(c, seqs=seqs, low=low, high=min(high, low + 3000), **new,
                pieces=rng.randint(1, min(2, seqs)), piece=_log(rng, 16, 300))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _State:
    pass


class _Inputs:
    """Seeded tensors on the GPU, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 53)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV)

    def rows(self, n, width):
        """n rows of width values whose channels differ in size, some by far, as a
        projection's do."""
        size = torch.exp(0.5 * self.normal(width)) * torch.where(
            torch.rand(width, generator=self.g, device=DEV) < 0.02, 12.0, 1.0)
        return self.normal(n, width) * size

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _lengths(c):
    """(contexts after the step, new rows) of the case's sequences, as lists."""
    n, lo, hi = c["seqs"], c["new"], c["most"]
    ctx = [c["high"] if n == 1 else c["low"] + (c["high"] - c["low"]) * i // (n - 1)
           for i in range(n)]
    new = [c["piece"] if i * c["pieces"] // n < (i + 1) * c["pieces"] // n
           else lo + i * 7 % (hi - lo + 1) for i in range(n)]
    return [max(a, b) for a, b in zip(ctx, new)], new


def _cdiv(a, b):
    return (a + b - 1) // b


def _table(npos, D):
    i = torch.arange(D // 2, device=DEV, dtype=torch.float64)
    a = torch.arange(npos, device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-2 * i / D)
    return a.cos().float(), a.sin().float()


def _flat(counts):
    """For runs of these lengths one after another: each element's run, and its place in it."""
    run = torch.repeat_interleave(torch.arange(counts.numel(), device=DEV), counts)
    return run, torch.arange(run.numel(), device=DEV) - (counts.cumsum(0) - counts)[run]


def prepare(case, seed):
    r, s, c = _Inputs(seed), _State(), case
    s.case, op, ps, n = c, c["op"], c["page"], c["seqs"]
    mix = r.order(n)
    ctx, new = (torch.tensor(x, device=DEV)[mix] for x in _lengths(c))
    s.have, s.new = (ctx - new).int(), new.int()
    rows = int(new.sum())
    s.max_rows = _cdiv(max(rows, 1), 8) * 8  # a captured step's batch has room to spare
    if op == "step":
        return _prepare_step(r, s, c, ctx)
    q, kv, D = c["qheads"], c["kvheads"], c["hdim"]
    s.ctx = ctx.int()
    s.start = torch.cat([new.new_zeros(1), new.cumsum(0)]).int()
    s.max_new, s.max_ctx = max(1, int(new.max())), int(ctx.max())
    # of each list the pages that are read or written; the other entries are stale ids
    s.max_pages = _cdiv(s.max_ctx, ps)
    j = torch.arange(s.max_pages, device=DEV)
    used = j < _cdiv(ctx, ps)[:, None]
    first = (s.have.long() if op == "append" else s.have.long() - c["window"] + 1)
    live = used & ((j + 1) * ps > first[:, None])
    if op == "attention":
        live |= used & (j * ps < c["sinks"])
    s.npages = max(1, int(live.sum()))
    s.pages = r.ints(0, s.npages, n, s.max_pages).int()
    s.pages[live] = r.order(s.npages).int()[:int(live.sum())]
    seq, at = _flat(new)
    if op == "append":
        s.pos, s.slot = (torch.full((s.max_rows,), -1, device=DEV, dtype=t)
                         for t in (torch.int32, torch.int64))
        p = s.have[seq].long() + at
        s.pos[:rows] = p.int()
        s.slot[:rows] = s.pages[seq, p // ps].long() * ps + p % ps
        s.qkv = r.rows(s.max_rows, (q + 2 * kv) * D)
        s.cos, s.sin = _table(s.max_ctx, D)
        s.q = torch.zeros(s.max_rows, q * D, device=DEV)
        s.k, s.v = (torch.zeros(s.npages * ps, kv * D, dtype=torch.float16, device=DEV)
                    for _ in range(2))
        return s
    # the first tokens' keys meet every query, and their values are small
    toward = r.normal(kv, D)
    s.q = (r.normal(s.max_rows, kv, q // kv, D) + toward[:, None]).view(s.max_rows, q * D)
    s.k = (r.rows(s.npages * ps, kv * D) * 0.5).half()
    s.v = r.rows(s.npages * ps, kv * D).half()
    seq, at = _flat(ctx.clamp(max=c["sinks"]))
    sink = s.pages[seq, at // ps].long() * ps + at % ps
    s.k[sink] += (toward * (6 / math.sqrt(D))).view(-1).half()
    s.v[sink] *= 0.05
    s.out = torch.zeros(s.max_rows, q * D, device=DEV)
    return s


def _prepare_step(r, s, c, ctx):
    ps, n = c["page"], c["seqs"]
    if n >= 16:  # some have ended since the last step
        s.have[5::16] = -1
    have = ctx - s.new.long()  # those that ended had positions too
    kept = _cdiv(c["sinks"], ps)
    before = (have - r.ints(0, 9, n)).clamp(min=0)  # the length of the step before
    gone = ((before - c["window"] + 1).clamp(min=0) // ps - kept).clamp(min=0)
    # a draft that was not accepted may have left a page more
    taken = _cdiv(have, ps) + (r.ints(0, 4, n) == 0).long() * (have > 0)
    s.max_pages = _cdiv(int(ctx.max()), ps) + 2
    j = torch.arange(s.max_pages, device=DEV)
    live = (j < taken[:, None]) & ((j < kept) | (j >= kept + gone[:, None]))
    held = int(live.sum())
    s.npages = int(_cdiv(ctx, ps).sum()) + 3 * n + 57
    ids = r.order(s.npages).int()
    s.pages = r.ints(0, s.npages, n, s.max_pages).int()
    s.pages[live] = ids[:held]
    s.free = torch.full((s.npages,), -1, device=DEV, dtype=torch.int32)
    begin = int(r.ints(0, s.npages, 1))
    s.free[(begin + torch.arange(s.npages - held, device=DEV)) % s.npages] = ids[held:]
    s.free_in = torch.tensor([begin, s.npages - held], device=DEV, dtype=torch.int32)
    s.held_in = torch.stack([taken, gone], 1).int().contiguous()
    s.outs = dict(
        free=torch.zeros(2, device=DEV, dtype=torch.int32), held=torch.zeros_like(s.held_in),
        start=torch.zeros(n + 1, device=DEV, dtype=torch.int32),
        ctx=torch.zeros(n, device=DEV, dtype=torch.int32),
        seq=torch.zeros(s.max_rows, device=DEV, dtype=torch.int32),
        pos=torch.zeros(s.max_rows, device=DEV, dtype=torch.int32),
        slot=torch.zeros(s.max_rows, device=DEV, dtype=torch.int64),
        taken=torch.zeros(n + 1, device=DEV, dtype=torch.int32),
        status=torch.zeros(4, device=DEV, dtype=torch.int32))
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_step(s):
    c, n, ps = s.case, s.case["seqs"], s.case["page"]
    kept = _cdiv(c["sinks"], ps)
    have, (taken, gone) = s.have.long(), s.held_in.long().unbind(1)
    begin, count = s.free_in.long().unbind(0)
    live = have >= 0
    add = torch.where(live, s.new.long(), 0)
    ctx = have.clamp(min=0) + add
    more = torch.where(live, (_cdiv(ctx, ps) - taken).clamp(min=0), 0)
    out = torch.minimum((have - c["window"] + 1).clamp(min=0) // ps, taken) - kept
    now = torch.where(live, torch.maximum(gone, out), 0)
    start, at = (torch.cat([x.new_zeros(1), x.cumsum(0)]) for x in (add, more))
    # pages given back, in order: those that fell out of the window, all of an ended one's
    j = torch.arange(s.max_pages, device=DEV)
    past = (j >= kept + gone[:, None]) & (j < kept + now[:, None])
    ended = ~live[:, None] & (j < taken[:, None]) & ((j < kept) | (j >= kept + gone[:, None]))
    back = s.pages[past | ended]
    i, k = torch.nonzero((j >= taken[:, None]) & (j < (taken + more)[:, None]), as_tuple=True)
    s.pages[i, k] = s.free[(begin + at[i] + k - taken[i]) % s.npages]
    s.free[(begin + count + torch.arange(back.numel(), device=DEV)) % s.npages] = back
    seq = torch.full((s.max_rows,), -1, device=DEV)
    pos, slot = seq.clone(), seq.clone()
    run, off = _flat(add)
    rows = run.numel()
    p = have[run] + off
    seq[:rows], pos[:rows] = run, p
    slot[:rows] = s.pages[run, p // ps].long() * ps + p % ps
    zero = begin * 0
    new = dict(free=torch.stack([(begin + at[n]) % s.npages, count - at[n] + back.numel()]),
               held=torch.stack([torch.where(live, taken + more, 0), now], 1), start=start,
               ctx=ctx, seq=seq, pos=pos, slot=slot, taken=at,
               status=torch.stack([zero, start[n], at[n], zero + back.numel()]))
    return dict({k: v.to(s.outs[k].dtype) for k, v in new.items()}, pages=s.pages, ring=s.free)


def _plain_rope(x, cos, sin, heads):
    a, b = x.view(x.shape[0], heads, 2, -1).unbind(2)
    c, s = cos[:, None], sin[:, None]
    return torch.stack([a * c - b * s, b * c + a * s], 2).view(x.shape)


def _plain_append(s):
    c = s.case
    q, kv, D = c["qheads"], c["kvheads"], c["hdim"]
    row = torch.nonzero(s.slot >= 0).view(-1)
    pos, slot = s.pos[row].long(), s.slot[row]
    a, k, v = s.qkv[row].split([q * D, kv * D, kv * D], 1)
    cos, sin = s.cos[pos], s.sin[pos]
    s.q[row] = _plain_rope(a, cos, sin, q)
    s.k[slot] = _plain_rope(k, cos, sin, kv).half()
    s.v[slot] = v.half()
    return dict(q=s.q, k=s.k, v=s.v)


def _plain_attention(s):
    c = s.case
    q, kv, D, ps, n = c["qheads"], c["kvheads"], c["hdim"], c["page"], c["seqs"]
    G, sinks, window, most = q // kv, c["sinks"], c["window"], s.max_new
    have, new, ctx = s.have.long(), s.new.long(), s.ctx.long()
    # the positions that a sequence's rows see: its first ones, and from lo on
    lo = (have - window + 1).clamp(min=sinks)[:, None]
    j = torch.arange(min(sinks + min(window, s.max_ctx) + most - 1, s.max_ctx), device=DEV)[None]
    t = torch.where(j < sinks, j, lo + j - sinks)
    real = t < ctx[:, None]
    t = torch.where(real, t, 0)
    at = torch.gather(s.pages.long(), 1, t // ps) * ps + t % ps
    k, v = (x[at].float().view(n, -1, kv, D).transpose(1, 2).contiguous() for x in (s.k, s.v))
    # the rows of a sequence side by side
    i = torch.arange(most, device=DEV)[None]
    p = have[:, None] + i
    row = torch.where(i < new[:, None], s.start[:-1].long()[:, None] + i, s.max_rows)
    x = torch.cat([s.q, s.q.new_zeros(1, q * D)])[row].view(n, most, kv, G, D)
    x = x.transpose(1, 2).reshape(n, kv, most * G, D)
    w = torch.matmul(x, k.transpose(2, 3).contiguous()).view(n, kv, most, G, -1) / math.sqrt(D)
    p, t, real = p[:, :, None], t[:, None], real[:, None]
    seen = real & (t <= p) & ((t > p - window) | (t < sinks))
    w = w.masked_fill(~seen[:, None, :, None], -math.inf)
    w = torch.exp(w - w.amax(4, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(w.view(n, kv, most * G, -1), v).view(n, kv, most, G, D)
    o = o / w.sum(4, keepdim=True)
    fine = i < new[:, None]
    s.out[row[fine]] = o.permute(0, 2, 1, 3, 4).reshape(n, most, q * D)[fine]
    return dict(out=s.out)


def _plain(s):
    return dict(step=_plain_step, append=_plain_append,
                attention=_plain_attention)[s.case["op"]](s)


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
    p, call, st, n = si.ptr, si.call, si.stream_handle(), c["seqs"]
    if op == "step":
        o = s.outs
        call("si_kv_step", n, p(s.have), p(s.new), s.max_rows, c["window"], c["sinks"], c["page"],
             s.npages, s.max_pages, p(s.pages), p(s.free), p(s.free_in), p(o["free"]),
             p(s.held_in), p(o["held"]), p(o["start"]), p(o["ctx"]), p(o["seq"]), p(o["pos"]),
             p(o["slot"]), p(o["taken"]), p(o["status"]), st)
        return dict(o, pages=s.pages, ring=s.free)
    shape = ctypes.byref(si.make_shape(32, c["qheads"], c["kvheads"], c["hdim"]))
    if op == "append":
        call("si_rope_kv_append_rows", shape, p(s.qkv), s.qkv.shape[1], s.max_rows,
             s.cos.shape[0], p(s.pos), p(s.slot), p(s.cos), p(s.sin), p(s.q), p(s.k), p(s.v),
             s.k.shape[0], st)
        return dict(q=s.q, k=s.k, v=s.v)
    sizes = (n, s.max_rows, s.max_new, s.max_ctx, c["window"], c["sinks"])
    need = si.lib().si_attention_rows_workspace(shape, *sizes)
    ws = _workspace(need)
    call("si_attention_rows", shape, p(s.q), *sizes, p(s.start), p(s.ctx), p(s.k), p(s.v),
         s.npages, c["page"], p(s.pages), s.max_pages, p(s.out), None, None, None, p(ws), need, st)
    return dict(out=s.out)


def run(s):
    return _own(s) if own else _plain(s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Every live cache row, input and output once; two operations per multiply and add of the
    two products, six per rotated pair."""
    c, op, ps = case, case["op"], case["page"]
    ctx, new = _lengths(c)
    rows = sum(new)
    if op == "step":  # lengths, states and starts; the rows' entries; ids from the ring to the list
        return dict(bytes=40.0 * len(new) + 16.0 * rows + 8.0 * sum(_cdiv(x, ps) for x in new),
                    flops=0.0)
    qd, kvd = c["qheads"] * c["hdim"], c["kvheads"] * c["hdim"]
    if op == "append":
        return dict(bytes=float(rows * (8 * qd + 12 * kvd + 4 * c["hdim"] + 12)),
                    flops=3.0 * rows * (qd + kvd))
    window, sinks = c["window"], c["sinks"]
    union = seen = 0
    for L, m in zip(ctx, new):
        if m:
            lo = max(0, L - m - window + 1)
            union += L - lo + min(sinks, lo)
            for p in range(L - m, L):
                lo = max(0, p - window + 1)
                seen += p + 1 - lo + min(sinks, lo)
    return dict(bytes=4.0 * kvd * union + 8.0 * rows * qd, flops=4.0 * seen * qd)


# ---------------------------------------------------------------------------
# the same in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def exact(case, seed):
    def tables(s):
        c, ps, N = s.case, s.case["page"], s.npages
        window, kept = c["window"], -(-c["sinks"] // ps)
        pages, ring = s.pages.tolist(), s.free.tolist()
        begin, count = s.free_in.tolist()
        start, ctx, seq, pos, slot, taken, held, back = [0], [], [], [], [], [0], [], []
        for i, (h, a) in enumerate(zip(s.have.tolist(), s.new.tolist())):
            t, g = s.held_in[i].tolist()
            if h < 0:
                back += pages[i][:min(kept, t)] + pages[i][kept + g:t]
                start.append(start[-1])
                taken.append(taken[-1])
                ctx.append(0)
                held.append([0, 0])
                continue
            out = g
            while kept + out < t and (kept + out + 1) * ps - 1 <= h - window:
                back.append(pages[i][kept + out])
                out += 1
            need = 0
            while (t + need) * ps < h + a:
                pages[i][t + need] = ring[(begin + taken[-1] + need) % N]
                need += 1
            for x in range(h, h + a):
                seq.append(i)
                pos.append(x)
                slot.append(pages[i][x // ps] * ps + x % ps)
            start.append(start[-1] + a)
            taken.append(taken[-1] + need)
            ctx.append(h + a)
            held.append([t + need, out])
        for k, x in enumerate(back):
            ring[(begin + count + k) % N] = x
        pad = [-1] * (s.max_rows - len(seq))
        new = dict(free=[(begin + taken[-1]) % N, count - taken[-1] + len(back)], held=held,
                   start=start, ctx=ctx, seq=seq + pad, pos=pos + pad, slot=slot + pad, taken=taken,
                   status=[0, len(seq), taken[-1], len(back)])
        new = {k: torch.tensor(v, dtype=s.outs[k].dtype, device=DEV) for k, v in new.items()}
        return dict(new, pages=torch.tensor(pages, dtype=torch.int32, device=DEV),
                    ring=torch.tensor(ring, dtype=torch.int32, device=DEV))

    c, op = case, case["op"]
    s = prepare(case, seed)
    if op == "step":
        return tables(s)
    q, kv, D, ps = c["qheads"], c["kvheads"], c["hdim"], c["page"]
    if op == "append":
        n = int(s.new.sum())
        pos, slot = s.pos[:n].long(), s.slot[:n]
        x = s.qkv[:n].double().view(n, q + 2 * kv, D)
        cos, sin = s.cos.double()[pos][:, None], s.sin.double()[pos][:, None]
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        y = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
        out, k, v = s.q.double(), s.k.double(), s.v.double()
        out[:n] = y[:, :q].reshape(n, -1)
        k[slot], v[slot] = y[:, q:q + kv].reshape(n, -1), x[:, q + kv:].reshape(n, -1)
        return dict(q=out, k=k, v=v)
    out = s.out.double().view(-1, q, D)
    qq, ids = s.q.double().view(-1, q, D), torch.arange(s.max_ctx, device=DEV)
    for i, (L, m, at) in enumerate(zip(s.ctx.tolist(), s.new.tolist(), s.start.tolist())):
        if not m:
            continue
        first = max(0, L - m - c["window"] + 1)
        t = ids[:L]
        t = t[(t >= first) | (t < c["sinks"])]
        rows = s.pages[i].long()[t // ps] * ps + t % ps
        k, v = s.k[rows].double(), s.v[rows].double()
        dist = torch.arange(L - m, L, device=DEV)[:, None] - t[None]
        hidden = (dist < 0) | ((dist >= c["window"]) & (t >= c["sinks"])[None])
        for h in range(q):
            g = slice(h // (q // kv) * D, (h // (q // kv) + 1) * D)
            w = qq[at:at + m, h] @ k[:, g].T.contiguous() / math.sqrt(D)
            out[at:at + m, h] = torch.softmax(w.masked_fill_(hidden, -math.inf), 1) @ v[:, g]
    return dict(out=out.view(-1, q * D))
